"""The objectives over logits on the device: errors that all rows share, which a bound per row cannot see, and
what happens at borders (clip bounds, infinite margins, NaN among the operands)."""
import numpy as np
import pytest
import torch

import objective_reference as R
from rustautograd_b200 import frontend as F
from rustautograd_b200 import losses

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def on_device(cuda):
    F.use(cuda, "cuda")


def put(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def get(t):
    return t.cpu().numpy()


@pytest.mark.parametrize("rows,v,std", [(4096, 50257, 2.5), (4096, 50257, 1.0), (4096, 131072, 2.5), (8192, 8192, 2.5), (16384, 2049, 2.5), (32768, 1000, 2.5),
                                        (65536, 96, 2.5)])
def test_row_sums_have_no_error_in_common(rows, v, std):
    # A loss is a sum of terms of both signs. The roundings of N rows (u = 6e-8 each) average out as 1 / sqrt(N); an error that
    # is the same in all of them does not. Allowed: 1e-8, a sixth of u, and four standard errors of the mean.
    g = torch.Generator("cuda").manual_seed(v + rows)
    x = torch.randn((rows, v), generator=g, device="cuda") * std
    _, stats = losses.token_log_prob(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), stats=True)
    off = []
    for a in range(0, rows, 1024):
        y = x[a:a + 1024].double()
        m = y.amax(-1, keepdim=True)
        assert torch.equal(stats[a:a + 1024, 0].double(), m[:, 0])
        off.append(stats[a:a + 1024, 1].double() / torch.exp(y - m).sum(-1) - 1)
    off = torch.cat(off)
    assert abs(off.mean().item()) <= 1e-8 + 4 * off.std().item() / rows ** 0.5, (off.mean().item(), off.std().item())


def test_clip_bounds_are_not_rounded():
    # A clipped token's term is the bound times the advantage, rounded once: half a step, 2^-24 relatively.
    from test_objectives_exactness import clipped_tokens
    for v in (8, 3000, 20000):
        x, lab, old, adv, want = clipped_tokens(np.random.default_rng(v), 512, v)
        one = torch.ones(512, device="cuda")
        for grad in (False, True):
            terms = get(losses.policy_loss(*put(x, lab, old, adv), one, clip_low=0.2, clip_high=0.28, grad=grad).terms)
            assert (np.abs(terms.astype("f8") - want) <= 2.0 ** -24 * (1 + 1e-6) * np.abs(want)).all(), v


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("smoothing", [0.0, 0.25, 1.0])
def test_infinite_margins(smoothing, dtype):
    from test_objectives_exactness import check_infinite_margins, infinite_margins
    for v, t in ((6, 3), (3000, 3)):
        x, lab, w, ref, seq = infinite_margins(dtype, v, t)
        for pairs, signs in (([0, 2], (np.inf, 0)), ([1, 2], (-np.inf, 0)), ([0, 1, 2], (np.inf, -np.inf, 0))):
            rows = pairs + [p + 3 for p in pairs]
            r = losses.preference_loss(*put(x[rows], lab[rows], w[rows], ref[rows]), beta=0.5, smoothing=smoothing)
            check_infinite_margins(get(r.loss), get(r.margins), get(r.grad), signs, seq, smoothing, np.finfo(dtype).eps / 2 * (v / 32 + 40 + 100))
            alone = losses.preference_loss(*put(x[rows], lab[rows], w[rows], ref[rows]), beta=0.5, smoothing=smoothing, grad=False)
            assert torch.equal(alone.loss, r.loss)
    # Long sequences, where a block takes a pair.
    x, lab = torch.zeros((2, 300, 4), device="cuda"), torch.zeros((2, 300), dtype=torch.int32, device="cuda")
    x[1, 7, 0] = -float("inf")
    r = losses.preference_loss(x, lab, torch.ones((2, 300), device="cuda"), torch.zeros(2, device="cuda"), smoothing=smoothing)
    assert r.loss.item() == (0 if smoothing == 0 else float("inf")) and r.margins.item() == float("inf")


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("v", [40, 3000, 70000])
def test_nan_among_the_operands_reaches_the_gradient(v, dtype):
    from test_objectives_exactness import check_nan_operands, nan_operands
    x, lab, good, bad = nan_operands(np.random.default_rng(v), v, dtype)
    for kl in (0.0, 0.1):
        def policy(o):
            r = losses.policy_loss(*put(x, lab, o["old"], o["adv"], o["w"]), ref_logp=put(o["ref"])[0] if kl else None, kl=kl)
            return [get(t) for t in r]
        check_nan_operands(policy(good), policy(bad), kl)
    # A = 0 and a ratio past the largest number: the bound counts, and the term and its gradient are 0.
    one = torch.ones(1, dtype=torch.from_numpy(x).dtype, device="cuda")
    r = losses.policy_loss(*put(x[:1], lab[:1]), one * -1000, one * 0, one)
    assert r.loss.item() == 0 and not r.grad.any()


@pytest.mark.parametrize("v", [8, 96, 1000, 2048])
def test_gradient_is_that_of_the_term_at_a_clip_bound(v):
    # Ratios within the roundings of a bound: a token is clipped in the gradient where it is in the term, by the ratio of the row's
    # statistics in double. Float logits; old values a few steps around the one that gives the bound.
    n, rng = 8192, np.random.default_rng(v)
    x = rng.normal(size=(n, v)).astype("float32")
    lab = rng.integers(0, v, n).astype("int32")
    dx, dl = put(x, lab)
    stats = get(losses.token_log_prob(dx, dl, stats=True)[1]).astype("f8")
    lp = (x[np.arange(n), lab].astype("f8") - stats[:, 0]) - np.log(stats[:, 1])
    up = np.arange(n) % 2 == 0
    edge = np.where(up, 1 + 0.28, 1 - 0.2)
    old = (lp - np.log(edge)).astype("float32")
    for _ in range(3):
        old = np.where(rng.random(n) < 0.5, np.nextafter(old, np.float32(-100)), old)
    ratio = np.exp(lp - old.astype("f8"))
    clipped, sure = np.where(up, ratio > edge, ratio < edge), np.abs(ratio - edge) > 1e-14
    adv = np.where(up, 1, -1).astype("float32")
    r = losses.policy_loss(dx, dl, *put(old, adv, np.ones(n, "float32")), clip_low=0.2, clip_high=0.28)
    assert 0.1 < clipped.mean() < 0.9 and sure.mean() > 0.99
    assert np.array_equal((get(r.grad) == 0).all(1)[sure], clipped[sure])


@pytest.mark.parametrize("v", [40, 3000])
def test_small_divergences_in_double(v):
    # A reference next to the policy: exp(d) - d - 1 = d^2 / 2 and its slope -d, by differences that cancel.
    n, rng = 64, np.random.default_rng(v)
    x, lab = rng.normal(size=(n, v)), rng.integers(0, v, n).astype("int32")
    lp = R.log_prob(x, lab)
    ref = (lp + rng.uniform(0.5, 2, n) * 10.0 ** rng.uniform(-7, -5, n)).astype("f8")
    d, u, zero = ref.astype(R.L) - lp, 2.0 ** -53, np.zeros(n)
    r = losses.policy_loss(*put(x, lab, lp.astype("f8"), zero, np.ones(n), ), ref_logp=put(ref)[0], kl=1.0)
    # d is off by what lp is: u (additions + 2.3 * 12 + 4 for the sum, 4 log s, 4 |lp|), below 300 u here; then expm1 and a difference.
    off = u * (v / 32 + 40 + 28 + 4 + 4 * 9 + 4 * 12) + 8 * u * np.abs(d)
    want = np.expm1(d) - d
    assert (np.abs(get(r.terms) - want) <= np.abs(d) * off).all()
    slope = get(r.grad)[np.arange(n), lab] / (1 - np.exp(lp.astype("f8")))
    assert (np.abs(slope + np.expm1(d)) <= off + 16 * u * np.abs(d)).all()


@pytest.mark.parametrize("v,k", [(33, 31), (96, 64), (1040, 1000), (3001, 1024), (40000, 1024)])
def test_distillation_terms_are_rounded_once(v, k):
    # Equal logits and equal entries: both sums are whole numbers, computed without rounding, and the term is log(v / k): half a
    # step of its own, 2^-24, with no rounding of the two logarithms (4.8e-7 of a term of 0.04).
    x, teacher = torch.full((5, v), 3.0, device="cuda"), torch.full((5, k), -2.0, device="cuda")
    index = torch.arange(k, dtype=torch.int32, device="cuda").flip(0).repeat(5, 1)
    for grad in (False, True):
        terms = get(losses.distillation_loss(x, index, teacher, torch.ones(5, device="cuda"), grad=grad).terms).astype("f8")
        assert (np.abs(terms - np.log(v / k)) <= 2.0 ** -24 * (1 + 1e-6) * np.log(v / k)).all(), (grad, terms)


def test_launch_counts():
    # What a program says it launches is what the direct calls launch (the nodes of their captured graphs); a step whose loss
    # nobody reads has no sum.
    import ctypes
    n, t, v = 4, 3, 50
    rng = np.random.default_rng(0)
    x, lab = rng.normal(size=(n, t, v)).astype("float32"), rng.integers(0, v, (n, t)).astype("int32")
    index, row, seq = rng.integers(0, v, (n, t, 5)).astype("int32"), np.ones((n, t), "float32"), np.ones(n, "float32")
    teacher = rng.normal(size=(n, t, 5)).astype("float32")
    dx, dl, di, dr, ds, dt = put(x, lab, index, row, seq, teacher)
    tx, tl, ti, tr, ts, tt = (F.tensor(a) for a in (x, lab, index, row, seq, teacher))
    cudart = ctypes.CDLL("libcudart.so.12")

    def nodes(call):
        call()
        g = torch.cuda.CUDAGraph(keep_graph=True)
        with torch.cuda.graph(g):
            call()
        count = ctypes.c_size_t()
        assert cudart.cudaGraphGetNodes(ctypes.c_void_p(g.raw_cuda_graph()), None, ctypes.byref(count)) == 0
        return count.value

    def launches(f):
        c = F.compile(f, (tx,), validate="none", device="cuda")
        c(tx)
        before = c._n.launches()
        c(tx)
        return c._n.launches() - before
    logp, policy = lambda x: F.nn.token_log_prob(x, tl), lambda x: F.nn.policy_loss(x, tl, tr, tr, tr)[0]
    preference, distill = lambda x: F.nn.preference_loss(x, tl, tr, ts)[0], lambda x: F.nn.distillation_loss(x, ti, tt, tr)[0]
    assert launches(logp) == nodes(lambda: losses.token_log_prob(dx, dl)) == 1
    for grad, of in ((False, lambda f: f), (True, F.value_and_grad)):
        assert launches(of(policy)) == nodes(lambda: losses.policy_loss(dx, dl, dr, dr, dr, grad=grad)) == 2
        assert launches(of(distill)) == nodes(lambda: losses.distillation_loss(dx, di, dt, dr, grad=grad)) == 2
        assert launches(of(preference)) == nodes(lambda: losses.preference_loss(dx, dl, dr, ds, grad=grad)) == 2 + grad
    assert launches(F.grad(policy)) == launches(F.grad(distill)) == 1 and launches(F.grad(preference)) == 3


def test_labels_that_count_are_checked():
    from test_objectives_exactness import check_labels
    check_labels("cuda")


def check_step(names, before, gpu, cpu, what):
    """A step's outputs (count, first and second moments, parameters, then the loss and what goes with it) against the interpreter's, each
    leaf at its own size. From zero moments the first one is a tenth of the gradient."""
    from helpers import max_rel
    from test_gpu_baseline_configs import TOL, check_gradient, check_parameter
    n = len(names)
    assert gpu[0] == cpu[0] == 1
    for k in range(n):
        check_gradient(f"{what}: mu {names[k]}", gpu[1 + k], cpu[1 + k])
        check_gradient(f"{what}: nu {names[k]}", gpu[1 + n + k], cpu[1 + n + k])
        check_parameter(f"{what}: {names[k]}", before[k], gpu[1 + 2 * n + k], cpu[1 + 2 * n + k], gpu[1 + k], gpu[1 + n + k], cpu[1 + k] / 0.1)
    assert len(gpu) > 1 + 3 * n
    for g, w in zip(gpu[1 + 3 * n:], cpu[1 + 3 * n:]):
        assert max_rel(g, w) <= TOL, (what, g, w)


def test_training_steps_against_the_interpreter(oracle):
    from helpers import np_of, triple
    from test_gpu_baseline_configs import leaf_paths
    from test_objectives import gpt_batches
    rng = np.random.default_rng(13)
    model = F.gpt.GPT(vocab=40, block=16, d=32, heads=4, layers=2)
    params, opt = model.init(F.random.key(0)), F.optim.adamw(1e-3)
    state, names = {"params": params, "opt": opt.init(params)}, leaf_paths(params)
    policy, preference, distill = gpt_batches(rng, 6, 16, 40, 5)
    for what, step, batch in (("policy", F.gpt.make_policy_step(model, opt, kl=0.05), policy), ("preference", F.gpt.make_preference_step(model, opt), preference),
                              ("distillation", F.gpt.make_distillation_step(model, opt, 2.0), distill)):
        c = F.compile(step, (state, batch), validate="none", device="cuda")
        leaves = [F.tensor(leaf) for leaf in F.flatten((state, batch))[0]]
        cpu = [np_of(o) for o in oracle.run_plan_blob(c.plan_blob(), [triple(leaf) for leaf in leaves])]
        gpu = [F.Tensor(o).numpy() for o in c._n.call([leaf._t for leaf in leaves])]
        before = [t.numpy() for t in F.tree_leaves(params)]
        check_step(names, before, gpu, cpu, what)
        # The check sees a gradient that is missing or off by a thousandth in any leaf, and an update that was left out.
        for k in range(len(names)):
            for wrong in (0.0, 1.001):
                with pytest.raises(AssertionError):
                    check_step(names, before, gpu, [a * np.float32(wrong) if j == 1 + k else a for j, a in enumerate(cpu)], what)
            with pytest.raises(AssertionError):
                check_step(names, before, [before[k] if j == 1 + 2 * len(names) + k else a for j, a in enumerate(gpu)], cpu, what)


def test_overwritten_logits_are_known_to_autograd():
    # exp keeps its result for its gradient; once that memory holds the loss's gradient, going back through it is refused.
    lab, w = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda")
    stats = losses.token_log_prob(torch.ones(4, 9, device="cuda"), lab, stats=True)[1]
    calls = [lambda x: losses.token_log_prob_grad(x, lab, stats, w, out=x), lambda x: losses.policy_loss(x, lab, -w, w, w, out=x),
             lambda x: losses.preference_loss(x.view(2, 2, 9), lab.view(2, 2), w.view(2, 2), w[:2], out=x.view(2, 2, 9)),
             lambda x: losses.distillation_loss(x, lab[:, None], w[:, None], w, out=x)]
    for call in calls:
        x = torch.zeros(4, 9, device="cuda", requires_grad=True)
        y = x.exp()
        losses.token_log_prob(y.detach(), lab)
        y.sum().backward(retain_graph=True)
        call(y.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("v", [5, 96, 3001, 40000])
def test_ends_of_the_temperature(v, dtype):
    # Cold: all of p and q at the largest logits, so a row whose teacher agrees costs nothing and one whose teacher does not costs the gap in
    # logits times T. Hot: p and q are uniform, the term is T^2 log(v / k) and the gradient T (1 / v - 1 / k at the entries).
    rng = np.random.default_rng(v)
    n, k = 6, 3
    x = rng.permuted(np.tile(np.arange(v) * (8.0 / v), (n, 1)), axis=1).astype(dtype)
    order = np.argsort(-x, 1)
    index = order[:, [0, 1, 2]].astype("int32")
    teacher = np.tile(np.array([5, 4, 3], dtype), (n, 1))
    teacher[3:] = teacher[3:, ::-1]  # the third largest is the teacher's choice
    dx, di, dt = put(x, index, teacher)
    one = torch.ones(n, dtype=dx.dtype, device="cuda")
    u, at = np.finfo(dtype).eps / 2, np.arange(n)
    gap = x[at, index[:, 0]].astype("f8") - x[at, index[:, 2]]
    for temp in (2.0 ** -60, 2.0 ** -20):
        for grad in (False, True):
            r = losses.distillation_loss(dx, di, dt, one, temperature=temp, grad=grad)
            terms = get(r.terms)
            assert not terms[:3].any() and (np.abs(terms[3:] / temp - gap[3:]) <= 8 * u * gap[3:]).all(), (temp, terms)
        g = get(r.grad)
        want = np.zeros((n, v))
        want[at[3:], index[3:, 0]], want[at[3:], index[3:, 2]] = temp, -temp
        # The logits next to the largest are 8 / v below it: T exp(-8 / (v T)) of gradient, the others a power of that factor each (their
        # sum is below twice the first). It is 0 in either type at 2^-60, 8e-98 in double at 2^-20 and v = 40000.
        assert (np.abs(g - want.astype(dtype)) <= 2 * temp * np.exp(-8.0 / (v * temp))).all(), temp
    for temp in (2.0 ** 30, 2.0 ** 60):
        for grad in (False, True):
            r = losses.distillation_loss(dx, di, dt, one, temperature=temp, grad=grad)
            # The logits are within 8 / T of each other: 8e-9 of a term at most, and the sum of v ones is off by its additions.
            want = np.log(v / k)
            off = u * (v / 32 + 40 + 4 * want) + 8.0 / temp
            assert (np.abs(get(r.terms) / temp / temp - want) <= off).all(), temp
        g = get(r.grad).astype("f8") / temp
        want = np.full((n, v), 1.0 / v)
        np.subtract.at(want, (at[:, None], index), 1.0 / k)
        assert (np.abs(g - want) <= (u * (v / 32 + 60) + 16.0 / temp) * np.maximum(np.abs(want), 1 / v)).all(), temp


@pytest.mark.parametrize("v", [6, 3000, 40000])
def test_nan_in_one_pair_stays_in_it(v):
    # A NaN or +inf logit, a NaN weight or reference: loss and that pair's margin and gradients are NaN, the other pairs' are as they were.
    rng = np.random.default_rng(v)
    x, lab = rng.normal(size=(6, 4, v)).astype("float32"), rng.integers(0, v, (6, 4)).astype("int32")
    w, ref = np.ones((6, 4), "float32"), np.zeros(6, "float32")
    good = losses.preference_loss(*put(x, lab, w, ref))
    assert torch.isfinite(good.grad).all()
    for what in ("nan", "inf", "weight", "reference"):
        bx, bw, br = x.copy(), w.copy(), ref.copy()
        if what in ("nan", "inf"):
            bx[4, 2, v // 2] = float(what)
        elif what == "weight":
            bw[4, 2] = np.nan
        else:
            br[4] = np.nan
        r = losses.preference_loss(*put(bx, lab, bw, br))
        assert torch.isnan(r.loss) and torch.isnan(r.margins[1]) and torch.equal(r.margins[[0, 2]], good.margins[[0, 2]]), what
        assert torch.isnan(r.grad[[1, 4]]).all() if what != "inf" else torch.isnan(r.grad[1]).all(), what
        assert torch.equal(r.grad[[0, 2, 3, 5]], good.grad[[0, 2, 3, 5]]), what
