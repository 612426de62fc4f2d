"""The objectives over logits on the CPU: the engine's operations in the interpreter against extended
precision, their gradients against differences, how they are recorded and refused, and the refusals of
the C ABI. (The device's kernels: test_gpu_objectives.py.)"""
import ctypes
import json

import numpy as np
import pytest

import objective_reference as R
import rustautograd_b200
from rustautograd_b200 import frontend as F

SIZES = [(1, 1), (3, 2), (5, 7), (4, 96), (6, 131)]
DTYPES = ["float32", "float64"]


@pytest.fixture
def cpu(oracle):
    F.use(oracle, "cpu")
    return oracle


def run(fn, *args, **kw):
    args = tuple(F.tensor(a) for a in args)
    return F.compile(fn, args, validate="none", **kw)(*args)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", R.KINDS)
def test_interpreter_against_extended_precision(cpu, kind, dtype):
    rng = np.random.default_rng(3)
    for rows, v in SIZES:
        x = R.logits(rng, rows, v, kind, dtype)
        lab = R.labels(rng, x)
        ct = rng.normal(size=rows).astype(dtype)
        lp, g = run(lambda x, c: F.value_and_grad(lambda x: ((F.nn.token_log_prob(x, F.tensor(lab)) * c).sum(), F.nn.token_log_prob(x, F.tensor(lab))),
                                                  has_aux=True)(x), x, ct)
        want_lp, want_g = R.token_log_prob(x, lab, ct, dtype, v)
        R.assert_within(lp[1].numpy(), want_lp, "logp")
        R.assert_within(g.numpy(), want_g, "gradient of logp")
        old, adv, w, ref = R.policy_inputs(rng, x, lab, dtype)
        for kl in (0.0, 0.1):
            def f(x):
                out = F.nn.policy_loss(x, F.tensor(lab), F.tensor(old), F.tensor(adv), F.tensor(w), F.tensor(ref) if kl else None, 0.2, 0.28, kl)
                return out[0], out[1:]
            (loss, (terms, logp)), g = run(F.value_and_grad(f, has_aux=True), x)
            for got, want, what in zip((loss, terms, logp, g), R.policy(x, lab, old, adv, w, ref, 0.2, 0.28, kl, dtype, v), ("loss", "terms", "logp", "gradient")):
                R.assert_within(got.numpy(), want, f"policy {what} {rows}x{v} kl {kl}")
        k = min(v, 5)
        index, teacher, w = R.teacher_inputs(rng, x, k, dtype)

        def h(x):
            out = F.nn.distillation_loss(x, F.tensor(index), F.tensor(teacher), F.tensor(w), 1.5)
            return out
        (loss, terms), g = run(F.value_and_grad(h, has_aux=True), x)
        for got, want, what in zip((loss, terms, g), R.distillation(x, index, teacher, w, 1.5, dtype, v), ("loss", "terms", "gradient")):
            R.assert_within(got.numpy(), want, f"distillation {what} {rows}x{v}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_preference_against_extended_precision(cpu, dtype):
    rng = np.random.default_rng(4)
    for b, t, v in [(2, 1, 3), (4, 5, 17), (6, 9, 96)]:
        x = R.logits(rng, b * t, v, "normal", dtype).reshape(b, t, v)
        lab = rng.integers(0, v, (b, t)).astype("int32")
        w = (rng.random((b, t)) < 0.7).astype(dtype)
        w[0] = 0  # a sequence whose mask leaves nothing
        ref = (-rng.random(b) * 3 * t).astype(dtype)

        def f(x):
            out = F.nn.preference_loss(x, F.tensor(lab), F.tensor(w), F.tensor(ref), 0.3, 0.1)
            return out[0], out[1:]
        (loss, (margins, logp)), g = run(F.value_and_grad(f, has_aux=True), x)
        for got, want, what in zip((loss, margins, logp, g), R.preference(x, lab, w, ref, 0.3, 0.1, dtype, v), ("loss", "margins", "logp", "gradient")):
            R.assert_within(got.numpy(), want, f"preference {what}")


@pytest.mark.parametrize("device", ["cpu", "cuda-plan"])
def test_gradients_against_differences(oracle, device):
    # The engine's own check: central differences of the float64 graph, on rg's plan and on the device's.
    F.use(oracle, device)
    rng = np.random.default_rng(5)
    x = rng.normal(size=(4, 3, 11))
    lab = F.tensor(rng.integers(0, 11, (4, 3)).astype("int32"))
    data = [F.tensor(rng.normal(size=(4, 3))) for _ in range(4)]
    index = F.tensor(rng.integers(0, 11, (4, 3, 4)).astype("int32"))
    teacher, ref = F.tensor(rng.normal(size=(4, 3, 4))), F.tensor(rng.normal(size=(4,)))
    losses = {
        "logp": lambda x: (F.nn.token_log_prob(x, lab) * data[0]).sum(),
        "policy": lambda x: F.nn.policy_loss(x, lab, data[0] - 2.0, data[1], data[2], data[3] - 2.0, kl=0.3)[0],
        "preference": lambda x: F.nn.preference_loss(x, lab, data[0], ref, smoothing=0.2)[0],
        "distillation": lambda x: F.nn.distillation_loss(x, index, teacher, data[1], 2.0)[0],
        # Scaled, and of logits that are themselves computed.
        "composed": lambda x: 3.0 * F.nn.distillation_loss(x * x, index, teacher, data[1])[0] - F.nn.token_log_prob(x + 1.0, lab).mean(),
    }
    for name, f in losses.items():
        c = F.compile(lambda x: F.value_and_grad(f)(x), (F.tensor(x),), validate="thorough")
        checks = {k["name"]: k["status"] for k in c.report["checks"]}
        assert c.report["status"] == "ok" and checks["grad_check"] == "pass" and checks["optimizer_equivalence"] == "pass", (name, c.report)


def test_equals_the_composition_it_stands_for(cpu):
    rng = np.random.default_rng(6)
    x, lab = rng.normal(size=(2, 5, 33)).astype("float32"), rng.integers(0, 33, (2, 5)).astype("int32")
    a = run(lambda x: F.value_and_grad(lambda x: -F.nn.token_log_prob(x, F.tensor(lab)).mean())(x), x)
    b = run(lambda x: F.value_and_grad(lambda x: F.nn.cross_entropy(x, F.tensor(lab)))(x), x)
    # Both are within the row bound of the exact value; ten rows of 33, so 2 * 60 u of a value below 8.
    assert abs(float(a[0]) - float(b[0])) <= 120 * 2.0 ** -24 * 8
    np.testing.assert_allclose(a[1].numpy(), b[1].numpy(), rtol=0, atol=120 * 2.0 ** -24)


def test_masked_rows_count_nothing_whatever_they_hold(cpu):
    rng = np.random.default_rng(7)
    x, lab = rng.normal(size=(4, 6, 9)).astype("float32"), rng.integers(0, 9, (4, 6)).astype("int32")
    w = (np.arange(6) < np.array([6, 3, 0, 5])[:, None]).astype("float32")
    bad = x.copy()
    bad[w == 0] = np.nan
    bad_lab = np.where(w == 0, -100, lab).astype("int32")
    other = {"old": rng.normal(size=(4, 6)).astype("float32"), "adv": rng.normal(size=(4, 6)).astype("float32")}
    bad_other = {k: np.where(w == 0, np.nan, v).astype("float32") for k, v in other.items()}
    index, teacher = rng.integers(0, 9, (4, 6, 3)).astype("int32"), rng.normal(size=(4, 6, 3)).astype("float32")
    ref = rng.normal(size=4).astype("float32")

    def all_of(x, lab, o):
        p = F.value_and_grad(lambda x: F.nn.policy_loss(x, F.tensor(lab), F.tensor(o["old"]), F.tensor(o["adv"]), F.tensor(w))[0])(x)
        q = F.value_and_grad(lambda x: F.nn.preference_loss(x, F.tensor(lab), F.tensor(w), F.tensor(ref))[0])(x)
        d = F.value_and_grad(lambda x: F.nn.distillation_loss(x, F.tensor(index), F.tensor(teacher), F.tensor(w))[0])(x)
        return p, q, d
    for good, masked in zip(F.tree_leaves(run(lambda x: all_of(x, lab, other), x)), F.tree_leaves(run(lambda x: all_of(x, bad_lab, bad_other), bad))):
        assert good.numpy().tobytes() == masked.numpy().tobytes()


def test_gradient_is_an_output_of_the_loss_step(oracle):
    # One pass over the logits: the gradient is a result of the loss's own step, not multiplied by the
    # loss's cotangent of 1, and a loss that is only evaluated has no such result.
    F.use(oracle, "cuda-plan")
    x, lab = F.zeros((3, 7)), F.zeros((3,), "int32")
    w = F.ones((3,))
    f = lambda x: F.nn.policy_loss(x, lab, w, w, w)[0]
    steps = json.loads(F.compile(F.value_and_grad(f), (x,), validate="none")._n.plan_summary())
    assert [s.get("op", "fused") for s in steps] == ["policy_loss"]
    c = F.compile(f, (x,), validate="none")
    assert [s.get("op", "fused") for s in json.loads(c._n.plan_summary())] == ["policy_loss"]
    assert c._n.output_shapes == [[]]


def test_refused_operands(cpu):
    x, lab = F.zeros((4, 3, 5)), F.zeros((4, 3), "int32")
    row, seq = F.zeros((4, 3)), F.zeros((4,))
    bad = [
        lambda: F.nn.token_log_prob(x, F.zeros((4, 2), "int32")),
        lambda: F.nn.token_log_prob(x, F.zeros((4, 3))),
        lambda: F.nn.token_log_prob(x.cast("int32"), lab),
        lambda: F.nn.token_log_prob(F.tensor(np.zeros((4, 0), "float32")), F.zeros((4,), "int32")),
        lambda: F.nn.policy_loss(x, lab, row, row, seq),
        lambda: F.nn.policy_loss(x, lab, row, row, F.tensor(np.zeros((4, 3)))),
        lambda: F.nn.policy_loss(x, lab, row, row, row, clip_low=-0.1),
        lambda: F.nn.policy_loss(x, lab, row, row, row, row, kl=float("nan")),
        lambda: F.nn.preference_loss(F.zeros((3, 3, 5)), F.zeros((3, 3), "int32"), F.zeros((3, 3)), F.zeros((3,))),
        lambda: F.nn.preference_loss(x, lab, row, row),
        lambda: F.nn.preference_loss(x, lab, row, seq, smoothing=1.5),
        lambda: F.nn.distillation_loss(x, F.zeros((4, 3, 2), "int32"), F.zeros((4, 3, 3)), row),
        lambda: F.nn.distillation_loss(x, F.zeros((4, 3, 2), "int32"), F.zeros((4, 3, 2)), row, temperature=0.0),
        lambda: F.nn.distillation_loss(x, F.zeros((4, 3, 1025), "int32"), F.zeros((4, 3, 1025)), row),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(Exception) as e:
            f()
        assert e.value.diagnostic["code"] == "OBJECTIVE_OPERANDS", k
    for kw in ({"kl": 0.1}, {"ref_logp": row}):
        with pytest.raises(ValueError):
            F.nn.policy_loss(x, lab, row, row, row, **kw)


def test_only_the_loss_is_differentiable(cpu):
    x, lab, w = F.zeros((2, 5)), F.zeros((2,), "int32"), F.ones((2,))
    for f in (lambda x: F.nn.policy_loss(x, lab, w, w, w)[1].sum(), lambda x: F.nn.distillation_loss(x, F.zeros((2, 1), "int32"), F.zeros((2, 1)), w)[1].sum(),
              lambda x: F.grad(lambda y: F.nn.token_log_prob(y, lab).sum())(x).sum()):
        with pytest.raises(Exception) as e:
            F.compile(lambda x: F.grad(f)(x), (x,), validate="none")
        assert e.value.diagnostic["code"] == "GRAD_UNSUPPORTED"
    # The other operands are data.
    g = run(lambda a: F.grad(lambda a: F.nn.policy_loss(x, lab, w, a, w)[0])(a), w)
    assert not g.numpy().any()


def test_in_control_flow_and_a_run(cpu):
    # The gradient of a loss inside a scan body, and a training run over batches.
    rng = np.random.default_rng(8)
    xs, lab = F.tensor(rng.normal(size=(3, 4, 7))), F.tensor(rng.integers(0, 7, 4).astype("int32"))
    w = F.tensor(rng.normal(size=7))

    def scanned(w):
        return F.scan(lambda c, x: (c + F.nn.token_log_prob(x * w, lab).sum(), None), F.tensor(np.float64(0.0)), xs)[0]

    def unrolled(w):
        return F.nn.token_log_prob(xs[0] * w, lab).sum() + F.nn.token_log_prob(xs[1] * w, lab).sum() + F.nn.token_log_prob(xs[2] * w, lab).sum()
    a, b = run(F.value_and_grad(scanned), w.numpy()), run(F.value_and_grad(unrolled), w.numpy())
    np.testing.assert_allclose(a[0].numpy(), b[0].numpy(), rtol=1e-13)
    np.testing.assert_allclose(a[1].numpy(), b[1].numpy(), rtol=0, atol=1e-12)


def gpt_batches(rng, n, t, v, k):
    tokens = rng.integers(0, v, (n, t + 1)).astype("int32")
    w = (np.arange(t) < rng.integers(1, t + 1, n)[:, None]).astype("float32")
    policy = {"tokens": tokens, "old_logp": (-rng.random((n, t)) * 4).astype("float32"), "ref_logp": (-rng.random((n, t)) * 4).astype("float32"),
              "advantages": rng.normal(size=(n, t)).astype("float32"), "weights": (w / w.sum()).astype("float32")}
    preference = {"tokens": tokens, "weights": w, "ref_logp": (-3.5 * w.sum(1)).astype("float32")}
    distill = {"tokens": tokens[:, :-1].copy(), "index": rng.integers(0, v, (n, t, k)).astype("int32"), "teacher": rng.normal(size=(n, t, k)).astype("float32"),
               "weights": policy["weights"]}
    return policy, preference, distill


@pytest.mark.parametrize("device", ["cpu", "cuda-plan"])
def test_gpt_training_steps(oracle, device):
    # The steps after pretraining, one after another on one model, as a program runs them.
    F.use(oracle, device)
    rng = np.random.default_rng(9)
    model = F.gpt.GPT(vocab=32, block=8, d=16, heads=2, layers=1)
    params = model.init(F.random.key(0))
    opt = F.optim.adamw(1e-3)
    state = {"params": params, "opt": opt.init(params)}
    policy, preference, distill = gpt_batches(rng, 4, 8, 32, 5)
    score = F.gpt.compile_scorer(model, params, F.tensor(policy["tokens"]))
    policy["old_logp"] = score(params, F.tensor(policy["tokens"])).numpy()
    for make, batch in ((F.gpt.make_policy_step(model, opt, kl=0.05), policy), (F.gpt.make_preference_step(model, opt), preference),
                        (F.gpt.make_distillation_step(model, opt, 2.0), distill)):
        c = F.compile(make, (state, batch), validate="basic")
        assert c.report.ok
        r = F.run(c, state, batch, steps=3)
        assert r.status == "completed" and all(np.isfinite(h).all() for h in r.history.values())
        state = r.state
    # The policy's first step starts at the sampling policy: no drift.
    first = F.run(F.compile(F.gpt.make_policy_step(model, opt, kl=0.05), ({"params": params, "opt": opt.init(params)}, policy), validate="none"),
                  {"params": params, "opt": opt.init(params)}, policy, steps=1)
    assert abs(first.history["aux.drift"][0]) <= 1e-6


# ---- the C ABI's refusals: every check below comes before any CUDA call or launch ----

class Logits(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("outer", ctypes.c_int64), ("inner", ctypes.c_int64), ("vocab", ctypes.c_int64),
                ("outer_stride", ctypes.c_int64), ("inner_stride", ctypes.c_int64), ("dtype", ctypes.c_int)]


class Gradient(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("outer_stride", ctypes.c_int64), ("inner_stride", ctypes.c_int64)]


class Policy(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("old_logp", "advantage", "weight", "ref_logp")] + [(n, ctypes.c_double) for n in ("clip_low", "clip_high", "kl")]


class Preference(ctypes.Structure):
    _fields_ = [("weight", ctypes.c_void_p), ("ref_logp", ctypes.c_void_p), ("beta", ctypes.c_double), ("smoothing", ctypes.c_double)]


class Distillation(ctypes.Structure):
    _fields_ = [("index", ctypes.c_void_p), ("teacher", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("entries", ctypes.c_int64), ("temperature", ctypes.c_double)]


def test_abi_refusals(product):
    lib = ctypes.CDLL(rustautograd_b200.LIBRARY)
    lib.rgc_last_error.restype = ctypes.c_char_p
    lib.rgc_preference_workspace.restype = ctypes.c_size_t
    fake = ctypes.c_void_p(1 << 20)  # never dereferenced

    def logits(**kw):
        f = dict(data=1 << 20, outer=4, inner=3, vocab=8, outer_stride=24, inner_stride=8, dtype=0)
        f.update(kw)
        return Logits(**f)

    def refused(rc, part):
        assert rc == -1 and part in lib.rgc_last_error(), (rc, lib.rgc_last_error())

    for kw, part in [({"dtype": 2}, b"dtype"), ({"outer": -1}, b"negative"), ({"vocab": 0}, b"vocab"), ({"vocab": 1 << 31}, b"vocab"),
                     ({"outer": 1 << 41}, b"too many rows"), ({"outer": 1 << 30, "inner": 1 << 30}, b"too many rows"), ({"inner_stride": -8}, b"strides")]:
        x = logits(**kw)
        refused(lib.rgc_token_log_prob(ctypes.byref(x), fake, fake, fake, None), part)
    refused(lib.rgc_token_log_prob(None, fake, fake, fake, None), b"null")
    x = logits()
    refused(lib.rgc_token_log_prob(ctypes.byref(x), fake, None, None, None), b"no output")
    p = Policy(fake, fake, fake, None, 0.2, 0.2, 0.0)
    for so, si, part in [(24, 7, b"overlap"), (16, 8, b"overlap"), (-24, 8, b"strides")]:
        g = Gradient(1 << 24, so, si)
        refused(lib.rgc_policy_loss(ctypes.byref(x), fake, ctypes.byref(p), fake, fake, None, ctypes.byref(g), None), part)
    g = Gradient((1 << 20) + 32, 24, 8)  # one row further in the logits' own memory
    refused(lib.rgc_policy_loss(ctypes.byref(x), fake, ctypes.byref(p), fake, fake, None, ctypes.byref(g), None), b"overlaps the logits")
    for field, value in [("clip_low", -0.1), ("clip_high", float("nan")), ("kl", float("inf"))]:
        q = Policy(fake, fake, fake, None, 0.2, 0.2, 0.0)
        setattr(q, field, value)
        refused(lib.rgc_policy_loss(ctypes.byref(x), fake, ctypes.byref(q), fake, fake, None, None, None), b"clip")
    need = lib.rgc_preference_workspace(ctypes.c_int64(4), ctypes.c_int64(3), 0)
    assert need == 4 * (3 * 12 + 3 * 2)
    pr = Preference(fake, fake, 0.1, 0.0)
    refused(lib.rgc_preference_loss(ctypes.byref(x), fake, ctypes.byref(pr), fake, None, None, None, fake, ctypes.c_size_t(need - 1), None), b"workspace")
    odd = logits(outer=3)
    refused(lib.rgc_preference_loss(ctypes.byref(odd), fake, ctypes.byref(pr), fake, None, None, None, fake, ctypes.c_size_t(need), None), b"even")
    pr.smoothing = 1.1
    refused(lib.rgc_preference_loss(ctypes.byref(x), fake, ctypes.byref(pr), fake, None, None, None, fake, ctypes.c_size_t(need), None), b"smoothing")
    for entries, temp, part in [(0, 1.0, b"entries"), (1025, 1.0, b"entries"), (4, 0.0, b"temperature"), (4, float("inf"), b"temperature")]:
        d = Distillation(fake, fake, fake, entries, temp)
        refused(lib.rgc_distillation_loss(ctypes.byref(x), ctypes.byref(d), fake, fake, None, None), part)


def test_call_refusals_without_a_gpu(product):
    import torch

    from rustautograd_b200 import losses
    with pytest.raises(TypeError, match="CUDA tensor"):
        losses.token_log_prob(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32))
    x = torch.zeros(4, 5, 6, 8)
    rows = lambda *a: losses._rows(*a)
    assert rows(x) == (120, 1, [8], [0])
    assert rows(x[:, :, :-1]) == (20, 5, [48], [8])
    assert rows(x[:, 0]) == (4, 6, [240], [8])
    assert rows(x[0, 0, 0]) == (1, 1, [0], [0])
    assert rows(x.transpose(0, 2)[:, :, 0]) == (6, 5, [8], [48])
    assert rows(x[0], torch.zeros(5, 7, 8)[:, :6]) == (5, 6, [48, 56], [8, 8])
    with pytest.raises(ValueError, match="two independent strides"):
        rows(x[:, :-1, :-1])
    with pytest.raises(ValueError, match="two independent strides"):
        rows(x[:, :, :-1], torch.zeros(4, 6, 5, 8)[:, :-1])
    with pytest.raises(ValueError, match="contiguous"):
        rows(x.transpose(2, 3))


def test_temperature_bounds(cpu):
    for temp in (2.0 ** -61, 2.0 ** 61, 1e-300, float("nan")):
        with pytest.raises(Exception) as e:
            F.nn.distillation_loss(F.zeros((4, 3, 8)), F.zeros((4, 3, 2), "int32"), F.zeros((4, 3, 2)), F.zeros((4, 3)), temperature=temp)
        assert e.value.diagnostic["code"] == "OBJECTIVE_OPERANDS"


def test_vouched_pointers_and_spans(product):
    """Vouching for the pointers leaves the other checks; rows that span too much are refused, not wrapped around."""
    lib = ctypes.CDLL(rustautograd_b200.LIBRARY)
    lib.rgc_last_error.restype = ctypes.c_char_p
    fake = ctypes.c_void_p(1 << 20)  # never dereferenced
    for dtype in (0, 1, 256, 257):
        for x, labels, part in [(Logits(1 << 20, 4, 3, 0, 24, 8, dtype), fake, b"vocab"), (Logits(1 << 20, 1 << 30, 1, 8, 1 << 40, 8, dtype), fake, b"span"),
                                (Logits(1 << 20, 4, 3, 8, 24, 8, dtype + 2), fake, b"dtype")]:
            assert lib.rgc_token_log_prob(ctypes.byref(x), labels, fake, fake, None) == -1 and part in lib.rgc_last_error()
        x, g = Logits(1 << 20, 1 << 30, 1, 8, 8, 8, dtype), Gradient(1 << 30, 1 << 40, 8)
        assert lib.rgc_token_log_prob_grad(ctypes.byref(x), fake, fake, fake, ctypes.byref(g), None) == -1 and b"span" in lib.rgc_last_error()
    x = Logits(1 << 20, 4, 3, 8, 24, 8, 256)
    assert lib.rgc_token_log_prob(ctypes.byref(x), None, fake, fake, None) == -1 and b"labels is null" in lib.rgc_last_error()
    odd = ctypes.c_void_p((1 << 20) + 2)
    assert lib.rgc_token_log_prob(ctypes.byref(x), odd, fake, fake, None) == -1 and b"aligned" in lib.rgc_last_error()
