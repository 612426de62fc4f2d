"""The objectives over logits on the device: the direct calls (rustautograd_b200.losses) and compiled
plans against extended precision, over sizes, types, strides and masks."""
import numpy as np
import pytest
import torch

import objective_reference as R
from rustautograd_b200 import frontend as F
from rustautograd_b200 import losses

pytestmark = pytest.mark.gpu

# Vocabularies around the widths the kernels change at, odd ones between; rows from one up.
SIZES = [(1, 1), (7, 2), (5, 31), (33, 65), (64, 96), (3, 129), (9, 257), (4, 1000), (17, 1009), (2, 1025), (5, 2052), (3, 4097), (6, 8190),
         (2, 16385), (3, 32000), (1, 50257), (2, 70001), (1, 131072), (1, 270001)]
DTYPES = ["float32", "float64"]


def adds(v):
    """Additions on the longest path of a row's sum: a 32nd of the row in one thread, then the joins."""
    return v / 32 + 40


@pytest.fixture(autouse=True)
def on_device(cuda):
    F.use(cuda, "cuda")


def put(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


def get(t):
    return t.cpu().numpy()


def check(got, want, names, what):
    for g, w, name in zip(got, want, names):
        R.assert_within(get(g), w, f"{name} of {what}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", SIZES)
def test_token_log_prob(rows, v, dtype):
    for kind in R.KINDS:
        rng = np.random.default_rng([rows, v, len(kind)])
        x = R.logits(rng, rows, v, kind, dtype)
        lab, ct = R.labels(rng, x), rng.normal(size=rows).astype(dtype)
        ct[rows // 2] = 0 if rows > 1 else ct[0]
        dx, dl, dc = put(x, lab, ct)
        logp, stats = losses.token_log_prob(dx, dl, stats=True)
        grad = losses.token_log_prob_grad(dx, dl, stats, dc)
        check((logp, grad), R.token_log_prob(x, lab, ct, dtype, adds(v)), ("logp", "gradient"), f"{rows}x{v} {kind}")
        assert torch.equal(losses.token_log_prob(dx, dl), logp)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", SIZES)
def test_policy_loss(rows, v, dtype):
    for kind in R.KINDS:
        rng = np.random.default_rng([rows, v, len(kind), 1])
        x = R.logits(rng, rows, v, kind, dtype)
        lab = R.labels(rng, x)
        old, adv, w, ref = R.policy_inputs(rng, x, lab, dtype)
        kl = 0.1 if len(kind) % 2 else 0.0
        want = R.policy(x, lab, old, adv, w, ref, 0.2, 0.28, kl, dtype, adds(v))
        bad, bad_lab = x.copy(), lab.copy()
        bad[w == 0] = np.nan
        bad_lab[w == 0] = -100
        args = put(bad, bad_lab, old, adv, w)
        kw = dict(ref_logp=put(ref)[0] if kl else None, clip_low=0.2, clip_high=0.28, kl=kl)
        r = losses.policy_loss(*args, **kw)
        check(r, want, r._fields, f"policy {rows}x{v} {kind}")
        alone = losses.policy_loss(*args, grad=False, **kw)
        assert alone.grad is None
        check(alone[:3], want, r._fields, f"policy without gradient {rows}x{v} {kind}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,t,v", [(2, 1, 1), (2, 3, 65), (4, 7, 96), (6, 37, 1009), (2, 5, 4097), (4, 3, 32000), (2, 2, 70001), (8, 300, 33)])
def test_preference_loss(b, t, v, dtype):
    rng = np.random.default_rng([b, t, v])
    for kind in ("normal", "banned"):
        x = R.logits(rng, b * t, v, kind, dtype)
        lab = R.labels(rng, x).reshape(b, t)
        x = x.reshape(b, t, v)
        w = (rng.random((b, t)) < 0.7).astype(dtype) * (0.5 if kind == "banned" else 1)
        if b > 2:
            w[1] = 0  # a sequence whose mask leaves nothing
        ref = (-rng.random(b) * 3 * t).astype(dtype)
        want = R.preference(x, lab, w, ref, 0.3, 0.1, dtype, adds(v))
        bad = x.copy()
        bad[w == 0] = np.nan
        args = put(bad, np.where(w == 0, -100, lab).astype("int32"), w.astype(dtype), ref)
        r = losses.preference_loss(*args, beta=0.3, smoothing=0.1)
        check(r, want, r._fields, f"preference {b}x{t}x{v} {kind}")
        alone = losses.preference_loss(*args, beta=0.3, smoothing=0.1, grad=False)
        check(alone[:3], want, r._fields, f"preference without gradient {b}x{t}x{v} {kind}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", SIZES)
def test_distillation_loss(rows, v, dtype):
    for kind, k, temp in (("normal", 8, 1.0), ("wide", 1, 2.0), ("banned", 33, 1.5), ("peaked", 300, 1.0)):
        rng = np.random.default_rng([rows, v, k])
        x = R.logits(rng, rows, v, kind, dtype)
        index, teacher, w = R.teacher_inputs(rng, x, k, dtype)
        if rows > 4:
            index[0] = index[0, 0]  # one index for every entry
        want = R.distillation(x, index, teacher, w, temp, dtype, adds(v))
        bad = x.copy()
        bad[w == 0] = np.nan
        args = put(bad, index, teacher, w)
        r = losses.distillation_loss(*args, temperature=temp)
        check(r, want, r._fields, f"distillation {rows}x{v} {kind} k {k}")
        alone = losses.distillation_loss(*args, temperature=temp, grad=False)
        check(alone[:2], want, r._fields, f"distillation without gradient {rows}x{v} {kind} k {k}")


def all_calls(x, lab, rng, dtype):
    """The four operators on (n, t, V) logits: a function of (logits, labels, out) to their outputs, gradients
    last in each, and what the outputs should be (None for the statistics)."""
    n, t, v = x.shape
    hx, hl = x.cpu().numpy().reshape(-1, v), lab.cpu().numpy().reshape(-1)
    old, adv, w, ref = R.policy_inputs(rng, hx, hl, dtype)
    index, teacher = rng.integers(0, v, (n * t, 6)).astype("int32"), rng.normal(size=(n * t, 6)).astype(dtype)
    seq = (-rng.random(n) * t).astype(dtype)
    want = [*R.token_log_prob(hx, hl, adv, dtype, adds(v)), *R.policy(hx, hl, old, adv, w, ref, 0.2, 0.28, 0.05, dtype, adds(v)),
            *R.preference(hx.reshape(n, t, v), hl.reshape(n, t), w.reshape(n, t), seq, 0.1, 0.0, dtype, adds(v)),
            *R.distillation(hx, index, teacher, w, 1.0, dtype, adds(v))]
    want.insert(1, None)
    dold, dadv, dw, dref = (a.reshape(n, t) for a in put(old, adv, w, ref))
    dindex, dteacher = (a.reshape(n, t, 6) for a in put(index, teacher))
    dseq = put(seq)[0]

    def go(x, lab, out=None):
        logp, stats = losses.token_log_prob(x, lab, stats=True)
        calls = [lambda: (logp, stats, losses.token_log_prob_grad(x, lab, stats, dadv, out=out)),
                 lambda: losses.policy_loss(x, lab, dold, dadv, dw, ref_logp=dref, clip_high=0.28, kl=0.05, out=out),
                 lambda: losses.preference_loss(x, lab, dw, dseq, out=out), lambda: losses.distillation_loss(x, dindex, dteacher, dw, out=out)]
        res = []
        for call in calls:
            *some, grad = call()
            res += [*some, grad if out is None else grad.clone()]
        return res
    return go, want


def check_all(got, want, what):
    for k, (g, w) in enumerate(zip(got, want)):
        if w is not None:
            R.assert_within(get(g), w, f"output {k} of {what}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 96, 1003, 8192, 33001])
def test_strides_alignment_and_neighbours(v, dtype):
    # Logits as positions of a longer output, from an odd address, with rows apart, and transposed; gradients
    # into views of every alignment whose surroundings stay as they were.
    rng = np.random.default_rng(v)
    n, t = 4, 5
    x = torch.from_numpy(R.logits(rng, n * t, v, "normal", dtype)).cuda().reshape(n, t, v)
    lab = torch.from_numpy(rng.integers(0, v, (n, t)).astype("int32")).cuda()
    go, want = all_calls(x, lab, rng, dtype)
    flat = torch.full((1 + (n * (t + 2) + 1) * (v + 3),), 7.0, dtype=x.dtype, device="cuda")
    views = {
        "plain": x,
        "shifted": torch.full((n, t + 1, v), 7.0, dtype=x.dtype, device="cuda")[:, :t],
        "odd address": flat[1:1 + n * t * v].view(n, t, v),
        "apart": flat[1:1 + n * (t + 2) * (v + 3)].view(n, t + 2, v + 3)[:, 1:t + 1, 2:v + 2],
        "transposed": torch.full((t, n, v), 7.0, dtype=x.dtype, device="cuda").transpose(0, 1),
    }
    for name, view in views.items():
        view.copy_(x)
        check_all(go(view, lab), want, f"{name} {v}")
        outs = {"like": view.clone() if name != "transposed" else torch.full_like(view, 3.0)}
        if name in ("plain", "shifted", "apart"):
            for first in range(4):
                base = torch.full((n, t + 2, v + 5), 3.0, dtype=x.dtype, device="cuda")
                outs[first] = base[:, 1:t + 1, first:v + first]
        for key, out in outs.items():
            check_all(go(view, lab, out), want, f"{name} to {key} {v}")
            if key != "like":
                base = out._base
                mark = torch.ones_like(base, dtype=torch.bool)
                mark[:, 1:t + 1, key:v + key] = False
                assert (base[mark] == 3.0).all(), (name, key)
    # Labels that are a view of something longer.
    wide = torch.zeros((n, t + 1), dtype=torch.int32, device="cuda")
    wide[:, 1:] = lab
    assert torch.equal(losses.token_log_prob(x, wide[:, 1:]), losses.token_log_prob(x, lab))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [7, 96, 1009, 8192, 40001, 300007])
def test_gradient_in_place_of_the_logits(v, dtype):
    rng = np.random.default_rng(v)
    n, t = 2, 3
    x = torch.from_numpy(R.logits(rng, n * t, v, "normal", dtype)).cuda().reshape(n, t, v)
    lab = torch.from_numpy(rng.integers(0, v, (n, t)).astype("int32")).cuda()
    w = torch.tensor([[1.0, 0.0, 0.5], [1.0, 1.0, 0.0]], dtype=x.dtype, device="cuda")
    old = torch.full((n, t), -2.0, dtype=x.dtype, device="cuda")
    seq = torch.zeros(n, dtype=x.dtype, device="cuda")
    index = torch.from_numpy(rng.integers(0, v, (n, t, 5)).astype("int32")).cuda()
    teacher = torch.from_numpy(rng.normal(size=(n, t, 5)).astype(dtype)).cuda()
    stats = losses.token_log_prob(x, lab, stats=True)[1]
    for name, f in {"logp": lambda x, out: losses.token_log_prob_grad(x, lab, stats, w, out=out), "policy": lambda x, out: losses.policy_loss(x, lab, old, w, w, out=out).grad,
                    "preference": lambda x, out: losses.preference_loss(x, lab, w, seq, out=out).grad,
                    "distillation": lambda x, out: losses.distillation_loss(x, index, teacher, w, out=out).grad}.items():
        want, y = f(x, None), x.clone()
        assert torch.equal(f(y, y), want), name


def test_many_rows_and_offsets_past_32_bits():
    # 2^31 elements and more: the last rows, the others without weight or uniform.
    rng = np.random.default_rng(0)
    v, rows = 50257, 43000
    x = torch.empty((rows, v), device="cuda")
    x[:-3] = 1.0
    tail = R.logits(rng, 3, v, "normal", "float32")
    x[-3:] = put(tail)[0]
    lab = rng.integers(0, v, rows).astype("int32")
    old, w, adv = np.full(rows, -9.0, "float32"), np.zeros(rows, "float32"), rng.normal(size=rows).astype("float32")
    w[-3:] = 0.5
    want = R.policy(tail, lab[-3:], old[-3:], adv[-3:], w[-3:], None, 0.2, 0.2, 0.0, "float32", adds(v))
    r = losses.policy_loss(x, *put(lab, old, adv, w), out=x)
    check((r.loss, r.terms[-3:], r.logp[-3:], r.grad[-3:]), want, r._fields, "the last rows")
    assert not r.grad[:-3].any() and not r.terms[:-3].any()
    del r
    x[:-3] = 1.0
    x[-3:] = put(tail)[0]
    logp, stats = losses.token_log_prob(x, put(lab)[0], stats=True)
    (want_logp, off), _ = R.token_log_prob(tail, lab[-3:], adv[-3:], "float32", adds(v))
    R.assert_within(get(logp[-3:]), (want_logp, off), "the last rows")
    # A uniform row: the statistics are exact up to the sum's rounding.
    assert (stats[:-3, 0] == 1.0).all() and ((stats[:-3, 1] - v).abs() <= v * (adds(v) + 4) * 2.0 ** -24).all()


def test_many_short_rows():
    # More rows than any grid, over the narrowest kernels.
    for v in (3, 96, 200):
        rng = np.random.default_rng(v)
        x = R.logits(rng, 70001, v, "normal", "float32")
        lab = R.labels(rng, x)
        old, adv, w, ref = R.policy_inputs(rng, x, lab, "float32")
        r = losses.policy_loss(*put(x, lab, old, adv, w), ref_logp=put(ref)[0], clip_high=0.28, kl=0.1)
        check(r, R.policy(x, lab, old, adv, w, ref, 0.2, 0.28, 0.1, "float32", adds(v)), r._fields, f"70001x{v}")


def test_empty_batches():
    for shape in ((0, 5), (3, 0, 5)):
        x = torch.empty(shape, device="cuda")
        row = torch.empty(shape[:-1], device="cuda")
        lab = torch.empty(shape[:-1], dtype=torch.int32, device="cuda")
        assert losses.token_log_prob(x, lab).shape == shape[:-1]
        r = losses.policy_loss(x, lab, row, row, row)
        assert r.loss.item() == 0 and r.grad.shape == shape
        many = torch.empty((*shape[:-1], 4), dtype=torch.int32, device="cuda")
        d = losses.distillation_loss(x, many, many.float(), row)
        assert d.loss.item() == 0 and d.terms.shape == shape[:-1]
    # Sequences without positions, and a batch whose weights are all zero.
    x, lab = torch.empty((2, 0, 5), device="cuda"), torch.empty((2, 0), dtype=torch.int32, device="cuda")
    p = losses.preference_loss(x, lab, torch.empty((2, 0), device="cuda"), torch.tensor([1.0, 3.0], device="cuda"), beta=0.5)
    h = 0.5 * ((0 - 1.0) - (0 - 3.0))
    assert abs(p.loss.item() - np.log1p(np.exp(-h))) <= 2.0 ** -23 and p.margins.item() == h and not p.logp.any()
    x, lab, zero = torch.full((4, 3, 50), float("nan"), device="cuda"), torch.full((4, 3), -100, dtype=torch.int32, device="cuda"), torch.zeros((4, 3), device="cuda")
    bad = torch.full((4, 3), float("nan"), device="cuda")
    r = losses.policy_loss(x, lab, bad, bad, zero)
    assert r.loss.item() == 0 and not r.grad.any() and not r.terms.any() and not r.logp.any()
    p = losses.preference_loss(x, lab, zero, torch.zeros(4, device="cuda"))
    assert not p.grad.any() and not p.margins.any()
    d = losses.distillation_loss(x, lab[..., None], bad[..., None], zero)
    assert d.loss.item() == 0 and not d.grad.any()


def test_nonfinite_rows_stay_apart():
    # A row of NaN, one with +inf and one of -inf give what the formulas give, and nothing reaches other rows.
    for v in (40, 3000, 70000):
        rng = np.random.default_rng(v)
        x = R.logits(rng, 6, v, "normal", "float32")
        clean = x.copy()
        x[1, v // 2] = np.nan
        x[2, v // 3] = np.inf
        x[4] = -np.inf
        lab, ct = np.full(6, v - 1, "int32"), np.ones(6, "float32")
        logp, stats = losses.token_log_prob(*put(x, lab), stats=True)
        grad = losses.token_log_prob_grad(*put(x, lab), stats, *put(ct))
        ok = [0, 3, 5]
        want = R.token_log_prob(clean[ok], lab[ok], ct[ok], "float32", adds(v))
        check((logp[ok], grad[ok]), want, ("logp", "gradient"), f"finite rows {v}")
        assert torch.isnan(logp[[1, 2, 4]]).all() and torch.isnan(grad[[1, 4]]).all()
        one = torch.ones(6, device="cuda")
        r = losses.policy_loss(*put(x, lab), logp.nan_to_num(-3.0), one, one)
        assert torch.isnan(r.loss) and torch.isfinite(r.grad[ok]).all() and torch.isnan(r.grad[[1, 4]]).all()
        index, teacher = np.tile(np.arange(3, dtype="int32"), (6, 1)), np.ones((6, 3), "float32")
        d = losses.distillation_loss(*put(x, index, teacher), one)
        assert torch.isfinite(d.grad[ok]).all() and torch.isnan(d.terms[[1, 2, 4]]).all()
        teacher[0] = np.nan  # not the same as absent
        assert torch.isnan(losses.distillation_loss(*put(x, index, teacher), one).terms[0])


def test_streams_graphs_and_repeats():
    rng = np.random.default_rng(11)
    cases = []
    for v in (96, 1009, 32000):
        x = torch.from_numpy(R.logits(rng, 24, v, "normal", "float32")).cuda().reshape(4, 6, v)
        lab = torch.from_numpy(rng.integers(0, v, (4, 6)).astype("int32")).cuda()
        cases.append((x, lab, all_calls(x, lab, rng, "float32")[0]))
    want = [go(x, lab) for x, lab, go in cases]
    torch.cuda.synchronize()
    # On two streams at once, and again: the same bits.
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for k, (x, lab, go) in enumerate(cases):
            with torch.cuda.stream(streams[k % 2]):
                got.append(go(x, lab))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    # Captured: two graphs replayed at the same time, on new contents of the same inputs.
    graphs, outs = [], []
    for x, lab, go in cases[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(go(x, lab))
        graphs.append(g)
    for x, _, _ in cases[:2]:
        x.mul_(0.5)
    torch.cuda.synchronize()
    for k, g in enumerate(graphs):
        with torch.cuda.stream(streams[k]):
            g.replay()
    torch.cuda.synchronize()
    for (x, lab, go), out in zip(cases, outs):
        assert all(torch.equal(p, q) for p, q in zip(out, go(x, lab)))


def test_refused_calls():
    x = torch.zeros((4, 3, 8), device="cuda")
    lab, row, seq = torch.zeros((4, 3), dtype=torch.int32, device="cuda"), torch.zeros((4, 3), device="cuda"), torch.zeros(4, device="cuda")
    for bad in (lambda: losses.token_log_prob(x.half(), lab), lambda: losses.token_log_prob(x, lab.long()), lambda: losses.token_log_prob(x, lab.cpu()),
                lambda: losses.policy_loss(x, lab, row.double(), row, row)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: losses.token_log_prob(x, lab[:2]), lambda: losses.token_log_prob(x.transpose(1, 2), torch.zeros((4, 8), dtype=torch.int32, device="cuda")),
                lambda: losses.policy_loss(x, lab, row, row, row, kl=0.1), lambda: losses.policy_loss(x, lab, row, row, row, ref_logp=row),
                lambda: losses.policy_loss(x, lab, row, row, row, clip_low=-1.0), lambda: losses.policy_loss(x, lab, row, row, row, grad=False, out=x),
                lambda: losses.policy_loss(x, lab, row, row, row, out=torch.empty((4, 3, 9), device="cuda")),
                lambda: losses.policy_loss(x[:, :2], lab[:, :2], row[:, :2], row[:, :2], row[:, :2], out=x[:, 1:]),
                lambda: losses.policy_loss(x, lab, row, row, row, out=torch.empty((3, 8), device="cuda").expand(4, 3, 8)),
                lambda: losses.preference_loss(x[:3], lab[:3], row[:3], seq[:3]), lambda: losses.preference_loss(x.view(12, 8), lab.view(12), row.view(12), seq),
                lambda: losses.preference_loss(x, lab, row, seq, smoothing=2.0), lambda: losses.distillation_loss(x, lab[..., None], row[..., None], row, temperature=0.0),
                lambda: losses.distillation_loss(x, lab[..., None].expand(4, 3, 1025), row[..., None].expand(4, 3, 1025), row),
                lambda: losses.distillation_loss(x, lab[..., None][..., :0], row[..., None][..., :0], row)):
        with pytest.raises(ValueError):
            bad()
    # A broadcast view of one row may be read.
    y = torch.arange(8.0, device="cuda").expand(4, 3, 8)
    assert torch.equal(losses.token_log_prob(y, lab), losses.token_log_prob(y.contiguous(), lab))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [11, 96, 4099, 33000])
def test_compiled_against_direct(v, dtype):
    # The same kernels through a plan: the bits of the direct calls.
    rng = np.random.default_rng(v)
    n, t = 4, 3
    x = R.logits(rng, n * t, v, "normal", dtype)
    lab = R.labels(rng, x)
    old, adv, w, ref = (a.reshape(n, t) for a in R.policy_inputs(rng, x, lab, dtype))
    x, lab = x.reshape(n, t, v), lab.reshape(n, t)
    index, teacher = rng.integers(0, v, (n, t, 5)).astype("int32"), rng.normal(size=(n, t, 5)).astype(dtype)
    seq = (-rng.random(n) * t).astype(dtype)
    ten = {k: F.tensor(a) for k, a in dict(lab=lab, old=old, adv=adv, w=w, ref=ref, index=index, teacher=teacher, seq=seq).items()}

    def f(x):
        p = F.value_and_grad(lambda x: (lambda o: (o[0], o[1:]))(F.nn.policy_loss(x, ten["lab"], ten["old"], ten["adv"], ten["w"], ten["ref"], kl=0.05)), has_aux=True)(x)
        q = F.value_and_grad(lambda x: (lambda o: (o[0], o[1:]))(F.nn.preference_loss(x, ten["lab"], ten["w"], ten["seq"])), has_aux=True)(x)
        d = F.value_and_grad(lambda x: F.nn.distillation_loss(x, ten["index"], ten["teacher"], ten["w"]), has_aux=True)(x)
        g = F.value_and_grad(lambda x: (F.nn.token_log_prob(x, ten["lab"]) * ten["adv"]).sum())(x)[1]
        return p, q, d, g, F.nn.token_log_prob(x, ten["lab"])
    c = F.compile(f, (F.tensor(x),), validate="none", device="cuda")
    got = [a.numpy() for a in F.tree_leaves(c(F.tensor(x)))]
    dx, dl, do, da, dw, dr, di, dt, ds = put(x, lab, old, adv, w, ref, index, teacher, seq)
    logp, stats = losses.token_log_prob(dx, dl, stats=True)
    want = [*losses.policy_loss(dx, dl, do, da, dw, ref_logp=dr, kl=0.05), *losses.preference_loss(dx, dl, dw, ds), *losses.distillation_loss(dx, di, dt, dw),
            losses.token_log_prob_grad(dx, dl, stats, da), logp]
    assert len(got) == len(want)
    for k, (a, b) in enumerate(zip(got, want)):
        assert a.tobytes() == get(b).tobytes(), k


def test_compiled_checks_and_training(oracle):
    # The engine's own checks on the device (differences of the float64 graph among them), and the GPT's
    # steps after pretraining against the interpreter.
    rng = np.random.default_rng(12)
    x, lab = rng.normal(size=(4, 3, 11)), F.tensor(rng.integers(0, 11, (4, 3)).astype("int32"))
    data = [F.tensor(rng.normal(size=(4, 3))) for _ in range(3)]
    index, teacher, ref = F.tensor(rng.integers(0, 11, (4, 3, 4)).astype("int32")), F.tensor(rng.normal(size=(4, 3, 4))), F.tensor(rng.normal(size=(4,)))
    for f in (lambda x: F.nn.policy_loss(x, lab, data[0] - 2.0, data[1], data[2])[0], lambda x: F.nn.preference_loss(x, lab, data[0], ref)[0],
              lambda x: F.nn.distillation_loss(x, index, teacher, data[1], 2.0)[0], lambda x: (F.nn.token_log_prob(x, lab) * data[0]).sum()):
        c = F.compile(lambda x: F.value_and_grad(f)(x), (F.tensor(x),), validate="thorough", device="cuda")
        assert c.report["status"] == "ok", c.report
    from helpers import max_rel, np_of, triple
    from test_objectives import gpt_batches
    model = F.gpt.GPT(vocab=40, block=16, d=32, heads=4, layers=2)
    params, opt = model.init(F.random.key(0)), F.optim.adamw(1e-3)
    state = {"params": params, "opt": opt.init(params)}
    policy, preference, distill = gpt_batches(rng, 6, 16, 40, 5)
    policy["old_logp"] = F.gpt.compile_scorer(model, params, F.tensor(policy["tokens"]), device="cuda")(params, F.tensor(policy["tokens"])).numpy()
    for step, batch in ((F.gpt.make_policy_step(model, opt, kl=0.05), policy), (F.gpt.make_preference_step(model, opt), preference),
                        (F.gpt.make_distillation_step(model, opt, 2.0), distill)):
        c = F.compile(step, (state, batch), validate="basic", device="cuda")
        leaves = [F.tensor(leaf) for leaf in F.flatten((state, batch))[0]]
        outs = c._n.call([leaf._t for leaf in leaves])
        cpu = [np_of(o) for o in oracle.run_plan_blob(c.plan_blob(), [triple(leaf) for leaf in leaves])]
        gpu = [F.Tensor(o).numpy() for o in outs]
        moments = len(gpu) - len(F.tree_leaves(params))
        for k, (a, b) in enumerate(zip(gpu, cpu)):
            # The framework's parity bound; updated parameters are held through the moments (a gradient
            # that is rounding noise can flip the sign of AdamW's first step, 2 lr).
            assert max_rel(a, b) <= 1e-4 or float(np.abs(a.astype("f8") - b).max()) <= 2.1e-3, (k, moments, max_rel(a, b))
        r = F.run(c, state, batch, steps=5)
        assert r.status == "completed" and r.steps == 5
        again = F.run(c, state, batch, steps=5)
        assert r.history == again.history
        state = r.state


@pytest.mark.parametrize("dtype", DTYPES)
def test_parts_of_a_row_without_any_logit(dtype):
    # Rows far below zero, with long stretches of -inf: whole lanes, warps and blocks hold nothing finite.
    for v in (70, 900, 3001, 20000, 70001, 300007):
        rng = np.random.default_rng(v)
        x = np.full((4, v), -np.inf, dtype)
        x[0, v // 2] = -5000.0                       # one logit: p = 1
        x[1, v - v // 3:] = rng.normal(size=v // 3) - 1000.0
        x[2, : v // 4] = rng.normal(size=v // 4) + 3000.0
        x[3, ::max(1, v // 7)] = -30000.0            # equal ones, far apart
        lab = R.labels(rng, x)
        old, adv, w, ref = R.policy_inputs(rng, x, lab, dtype)
        w = np.full(4, 0.25, dtype)
        check(losses.policy_loss(*put(x, lab, old, adv, w), clip_high=0.28), R.policy(x, lab, old, adv, w, ref, 0.2, 0.28, 0.0, dtype, adds(v)),
              ("loss", "terms", "logp", "grad"), f"sparse {v}")
        logp, stats = losses.token_log_prob(*put(x, lab), stats=True)
        grad = losses.token_log_prob_grad(*put(x, lab), stats, *put(adv))
        check((logp, grad), R.token_log_prob(x, lab, adv, dtype, adds(v)), ("logp", "grad"), f"sparse {v}")
        index, teacher = lab[:, None].copy(), np.zeros((4, 1), dtype)
        d = losses.distillation_loss(*put(x, index, teacher, w))
        check(d, R.distillation(x, index, teacher, w, 1.0, dtype, adds(v)), d._fields, f"sparse {v}")


# Vectors of 16 bytes to a row, around the numbers that the kernels for short rows and the blocks' sizes change at.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vectors", [8, 9, 16, 24, 25, 32, 50, 64, 100, 128, 150, 192, 193, 256, 300, 320, 321, 384, 385, 512, 513, 640, 641, 1025, 1449, 2049, 2897, 5793])
def test_widths_between_the_variants(vectors, dtype):
    v, rows = vectors * 16 // np.dtype(dtype).itemsize, 11
    rng = np.random.default_rng([vectors, len(dtype)])
    x = R.logits(rng, rows, v, "normal", dtype)
    lab = R.labels(rng, x)
    old, adv, w, ref = R.policy_inputs(rng, x, lab, dtype)
    w[3] = 0
    bad = x.copy()
    bad[w == 0] = np.nan
    want = R.policy(x, lab, old, adv, w, ref, 0.2, 0.28, 0.05, dtype, adds(v))
    r = losses.policy_loss(*put(bad, lab, old, adv, w), ref_logp=put(ref)[0], clip_low=0.2, clip_high=0.28, kl=0.05)
    check(r, want, r._fields, f"policy {rows} x {vectors} vectors")
    k = min(v, 13)
    index, teacher, w = R.teacher_inputs(rng, x, k, dtype)
    bad = x.copy()
    bad[w == 0] = np.nan
    want = R.distillation(x, index, teacher, w, 1.5, dtype, adds(v))
    r = losses.distillation_loss(*put(bad, index, teacher, w), temperature=1.5)
    check(r, want, r._fields, f"distillation {rows} x {vectors} vectors")
    logp, stats = losses.token_log_prob(*put(x, lab), stats=True)
    grad = losses.token_log_prob_grad(*put(x, lab), stats, *put(adv))
    check((logp, grad), R.token_log_prob(x, lab, adv, dtype, adds(v)), ("logp", "gradient"), f"{rows} x {vectors} vectors")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [3, 96, 700, 2051, 5001, 20000])
@pytest.mark.parametrize("k", [2, 5, 16, 32, 33, 64, 65, 257, 1024])
def test_numbers_of_teacher_entries(k, v, dtype):
    rng = np.random.default_rng([k, v])
    rows = 9
    x = R.logits(rng, rows, v, "normal", dtype)
    index, teacher, w = R.teacher_inputs(rng, x, k, dtype)
    w[:3] = 0.5
    index[0] = rng.integers(0, 2, k)          # the same index many times
    index[1, -1] = index[1, 0]                # the first and the last entry
    index[2] = 2 * v                          # past the vocabulary: its last element
    want = R.distillation(x, index, teacher, w, 0.7, dtype, adds(v))
    args = put(x, index, teacher, w)
    r = losses.distillation_loss(*args, temperature=0.7)
    check(r, want, r._fields, f"distillation {rows}x{v} k {k}")
    alone = losses.distillation_loss(*args, temperature=0.7, grad=False)
    check(alone[:2], want, r._fields, f"distillation without gradient {rows}x{v} k {k}")
    within = losses.distillation_loss(*args, temperature=0.7, out=args[0])
    assert torch.equal(args[0], r.grad) and torch.equal(within.terms, r.terms)


@pytest.mark.parametrize("b,t,v", [(40, 3, 5), (34, 1, 33), (6, 700, 9), (2, 257, 40), (70, 300, 3)])
def test_preferences_of_many_pairs_and_long_sequences(b, t, v):
    rng = np.random.default_rng([b, t, v])
    x = R.logits(rng, b * t, v, "normal", "float32")
    lab = R.labels(rng, x).reshape(b, t)
    x = x.reshape(b, t, v)
    w = ((rng.random((b, t)) < 0.7) / t).astype("float32")
    ref = (-rng.random(b) * 3).astype("float32")
    want = R.preference(x, lab, w, ref, 0.3, 0.1, "float32", adds(v))
    args = put(x, lab, w, ref)
    r = losses.preference_loss(*args, beta=0.3, smoothing=0.1)
    check(r, want, r._fields, f"preference {b}x{t}x{v}")
    again = losses.preference_loss(*args, beta=0.3, smoothing=0.1)
    assert all(torch.equal(p, q) for p, q in zip(r, again))


@pytest.mark.parametrize("v", [96, 5000])
def test_wide_and_tiny_doubles(v):
    """Doubles whose exponentials leave the normal range, and rows a constant apart: the polynomial's ends."""
    rng = np.random.default_rng(v)
    x = rng.normal(size=(6, v))
    x[0] *= 400
    x[1] = -rng.random(v) * 745
    x[2] = np.where(rng.random(v) < 0.5, -1e308, 0)
    x[3] = 1e15 + rng.integers(0, 64, v)
    x[4, 1:] = -709.0 + rng.random(v - 1)
    x[5] = np.linspace(-708, 0, v)
    lab, ct = np.argmax(x, 1).astype("int32"), np.ones(6)
    lab[5] = 0
    logp, stats = losses.token_log_prob(*put(x, lab), stats=True)
    grad = losses.token_log_prob_grad(*put(x, lab), stats, *put(ct))
    check((logp, grad), R.token_log_prob(x, lab, ct, "float64", adds(v)), ("logp", "gradient"), f"doubles {v}")


def test_entry_counts_in_turn():
    """More entries, fewer, and more again: the shared memory of the first call is still there for the third."""
    rng = np.random.default_rng(9)
    x, w = rng.normal(size=(9, 96)), np.full(9, 0.5)
    for k in (1024, 600, 1024, 7, 700):
        index, teacher = rng.integers(0, 96, (9, k)).astype("int32"), rng.random((9, k)) * 3
        r = losses.distillation_loss(*put(x, index, teacher, w))
        check(r, R.distillation(x, index, teacher, w, 1.0, "float64", adds(96)), r._fields, f"{k} entries")


def test_first_calls_inside_a_capture():
    """A process whose very first calls are captured: nothing they look up or load ends the capture."""
    import subprocess
    import sys

    script = """
import torch
from rustautograd_b200 import losses
x = torch.randn(6, 40, 2500, device="cuda")
y = torch.randn(6, 40, 200, device="cuda", dtype=torch.float64)
lab = torch.randint(0, 200, (6, 40), device="cuda", dtype=torch.int32)
w = torch.rand(6, 40, device="cuda")
seq = torch.rand(6, device="cuda", dtype=torch.float64)
index = torch.randint(0, 2500, (6, 40, 70), device="cuda", dtype=torch.int32)
teacher = torch.rand(6, 40, 70, device="cuda")
torch.cuda.synchronize()
calls = lambda: (losses.policy_loss(x, lab, -w, w, w), losses.preference_loss(y, lab, w.double(), seq), losses.distillation_loss(x, index, teacher, w),
                 losses.token_log_prob(y, lab, stats=True))
s = torch.cuda.Stream()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    got = calls()
g.replay()
torch.cuda.synchronize()
for a, b in zip(got, calls()):
    assert all(torch.equal(p, q) for p, q in zip(a, b))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr[-2000:]
