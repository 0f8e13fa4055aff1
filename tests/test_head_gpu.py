"""The language-model head on the GPU against plain forms in 64 bits.

Tolerances.  u is half a unit in the last place of the result's type (2^-24,
2^-11, 2^-8) and S its smallest positive number; a result is rounded to its
type once, so u * |value| + S covers that rounding.  The 32-bit arithmetic
before it adds, per operator, what the tests below derive: a sum of n terms,
however ordered, is off by at most n * 2^-24 * sum |terms|.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float32: E, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
S = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


@pytest.fixture(scope="module")
def zc():
    import zpu_b200
    zpu_b200.check(zpu_b200.lib().zpucuda_init(0))
    return zpu_b200


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def strided(t, pitch=0, shift=0):
    """The same values at another row pitch and start."""
    if not pitch and not shift:
        return t
    wide = torch.full((t.shape[0], t.shape[1] + pitch + shift), float("nan") if t.is_floating_point() else 99,
                      dtype=t.dtype, device=t.device)
    v = wide[:, shift:shift + t.shape[1]]
    v.copy_(t)
    return v


def within(got, want, tol, what=""):
    d = (got.double() - want).abs()
    ok = (d <= tol) | (got.double() == want) | (got.isnan() & want.isnan())
    if not bool(ok.all()):
        i = (~ok).nonzero()[0].tolist()
        raise AssertionError("%s: %d of %d off, first at %s: %r, %r is wanted within %r" % (
            what, int((~ok).sum()), ok.numel(), i, float(got[tuple(i)]), float(want[tuple(i)]),
            float(tol.expand_as(want)[tuple(i)])))


# ------------------------------------------------------------- layer norm
def ref_norm(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xhat = (x - mean) * rstd
    g = 1.0 if gamma is None else gamma.double()
    b = 0.0 if beta is None else beta.double()
    return xhat * g + b, mean, rstd, xhat, g, b


NORM_SIZES = [(1, 1), (3, 2), (5, 7), (2, 31), (4, 32), (7, 33), (300, 64), (9, 102), (2, 255), (3, 256), (1, 257), (65, 784),
              (33, 1000), (17, 1024), (3, 1025), (5, 2047), (4, 4096), (2, 4097), (3, 5003), (2, 8192), (2, 10007),
              (3, 16384), (2, 20480), (1, 32771), (2, 65536)]


def norm_inputs(rows, cols, t, wt, seed=1, pitch=0, shift=0, offset=0.0):
    g = gen(seed)
    x = (normal(g, rows, cols) * torch.exp(0.5 * normal(g, rows, 1)) + offset).to(TYPES[t])
    gamma = (1 + 0.2 * normal(g, cols)).to(TYPES[wt])
    beta = (0.1 * normal(g, cols)).to(TYPES[wt])
    return strided(x, pitch, shift), gamma, beta, g


def check_norm(zc, x, gamma, beta, eps=1e-5, **kw):
    y, mean, rstd = zc.layer_norm(x, gamma, beta, eps=eps, stats=True, **kw)
    want, m, r, xhat, g, b = ref_norm(x, gamma, beta, eps)
    n, u = x.shape[1], U[x.dtype]
    mag = x.double().abs().mean(1, keepdim=True)
    # the mean is a sum of n / 1 terms in chains no longer than n; the deviation inherits its error twice over
    chain = min(n, 160) + 8  # no thread adds more than n / 256 + 10 terms, and n <= 65536 here
    tm = chain * E * mag
    within(mean, m[:, 0], tm[:, 0] + 2 * E * m[:, 0].abs(), "mean")
    dev = tm + 2 * E * x.double().abs().amax(1, keepdim=True)  # of each x - mean
    tr = r * (chain * E + 2 * r * dev)
    within(rstd, r[:, 0], tr[:, 0], "rstd")
    t32 = (g * (r * dev + xhat * (tr / r)) if torch.is_tensor(g) else r * dev + xhat * (tr / r)).abs()
    t32 = t32 + 4 * E * ((xhat * g).abs() + (b.abs() if torch.is_tensor(b) else 0))
    within(y, want, t32 + u * (want.abs() + t32) + S[x.dtype], "y")
    return y


@pytest.mark.parametrize("t,wt", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16"),
                                  ("f32", "bf16")])
@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_layer_norm(zc, rows, cols, t, wt):
    x, gamma, beta, _ = norm_inputs(rows, cols, t, wt)
    check_norm(zc, x, gamma, beta)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("pitch,shift", [(1, 0), (8, 0), (3, 1), (16, 8), (5, 2)])
@pytest.mark.parametrize("cols", [64, 1000, 1001, 8192])
def test_layer_norm_strides(zc, cols, pitch, shift, t):
    x, gamma, beta, _ = norm_inputs(5, cols, t, "f32", pitch=pitch, shift=shift)
    y = check_norm(zc, x, gamma, beta)
    assert torch.equal(y, zc.layer_norm(x.contiguous(), gamma, beta))
    out = strided(torch.zeros_like(x.contiguous()), 7, 3)
    assert torch.equal(zc.layer_norm(x, gamma, beta, out=out), y)
    again = x.clone(memory_format=torch.contiguous_format)
    assert torch.equal(zc.layer_norm(again, gamma, beta, out=again), y)
    odd = torch.empty(cols + 1, device="cuda")[1:].copy_(gamma)  # weights off the vector grid
    assert torch.equal(zc.layer_norm(x, odd, beta), y)


def test_layer_norm_without_weights_and_far_from_zero(zc):
    for gamma, beta in ((True, False), (False, True), (False, False)):
        x, g, b, _ = norm_inputs(6, 777, "f32", "f32")
        check_norm(zc, x, g if gamma else None, b if beta else None)
    x, g, b, _ = norm_inputs(6, 4096, "f32", "f32", offset=1000.0)  # the variance is not a difference of squares
    check_norm(zc, x, g, b)
    x = torch.full((2, 300), 7.0, device="cuda")  # a constant row: 0 / sqrt(eps)
    y, mean, rstd = zc.layer_norm(x, eps=1e-5, stats=True)
    assert torch.equal(y, torch.zeros_like(x)) and bool((mean == 7).all())
    within(rstd, torch.full((2,), 1e-5, device="cuda").double() ** -0.5, torch.tensor(1e-3, device="cuda").double())


def test_layer_norm_keeps_nan_in_its_row(zc):
    x, g, b, _ = norm_inputs(64, 1024, "bf16", "f32")
    want = zc.layer_norm(x, g, b)
    x[5, 17], x[9, 3] = float("nan"), float("inf")
    y = zc.layer_norm(x, g, b)
    bad = torch.zeros(64, dtype=torch.bool, device="cuda")
    bad[5] = bad[9] = True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], want[~bad])


def check_norm_grad(zc, rows, cols, t, wt, pitch=0, shift=0, offset=0.0, weighted=True):
    x, gamma, _, g = norm_inputs(rows, cols, t, wt, pitch=pitch, shift=shift, offset=offset)
    if not weighted:
        gamma = None
    dy = strided((0.01 * normal(g, rows, cols)).to(TYPES[t]), pitch, shift)
    _, mean, rstd, _, gm, _ = ref_norm(x, gamma, None, 1e-5)
    mean, rstd = mean[:, 0].float(), rstd[:, 0].float()
    dx, dgamma, dbeta = zc.layer_norm_grad(dy, x, mean, rstd, gamma)
    d, r = dy.double(), rstd.double()[:, None]
    xhat = (x.double() - mean.double()[:, None]) * r
    exhat = 3 * E * (xhat.abs() + r * (x.double().abs() + mean.double().abs()[:, None]))  # of the 32-bit xhat
    gg = d * gm
    a, b = gg.mean(1, keepdim=True), (gg * xhat).mean(1, keepdim=True)
    want = r * (gg - a - xhat * b)
    chain = min(cols, 300) + 12
    ta = chain * E * gg.abs().mean(1, keepdim=True)
    tb = chain * E * (gg * xhat).abs().mean(1, keepdim=True) + (gg.abs() * exhat).mean(1, keepdim=True)
    t32 = r * (ta + xhat.abs() * tb + exhat * b.abs() + 6 * E * (gg.abs() + a.abs() + (xhat * b).abs()))
    u = U[x.dtype]
    within(dx, want, t32 + u * (want.abs() + t32) + S[x.dtype], "dx")
    n, uw = rows + 8, U[dgamma.dtype]
    for got, term, more, what in ((dgamma, d * xhat, (d.abs() * exhat).sum(0), "dgamma"), (dbeta, d, 0.0, "dbeta")):
        w = term.sum(0)
        tt = n * E * term.abs().sum(0) + more
        within(got, w, tt + uw * (w.abs() + tt) + S[got.dtype], what)
    return dy, x, mean, rstd, gamma, dx, dgamma, dbeta


@pytest.mark.parametrize("t,wt", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols", NORM_SIZES + [(1000, 10), (4097, 130), (700, 4096), (2500, 33)])
def test_layer_norm_grad(zc, rows, cols, t, wt):
    check_norm_grad(zc, rows, cols, t, wt)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("pitch,shift", [(1, 0), (8, 0), (3, 1)])
@pytest.mark.parametrize("cols", [65, 1024, 4099])
def test_layer_norm_grad_strides(zc, cols, pitch, shift, t):
    dy, x, mean, rstd, gamma, dx, dgamma, dbeta = check_norm_grad(zc, 37, cols, t, "f32", pitch, shift, offset=3.0)
    for k in (0, 1):  # in place of dy, of x
        a = [dy.clone(memory_format=torch.contiguous_format), x.clone(memory_format=torch.contiguous_format)]
        got = zc.layer_norm_grad(a[0], a[1], mean, rstd, gamma, out=a[k])
        assert got[0].data_ptr() == a[k].data_ptr()
        flat = zc.layer_norm_grad(dy.contiguous(), x.contiguous(), mean, rstd, gamma)
        assert all(torch.equal(p, q) for p, q in zip(got, flat))
    check_norm_grad(zc, 37, cols, t, "f32", pitch, shift, weighted=False)


def test_layer_norm_grad_against_differences(zc):
    """The gradient of sum(dy * y) in 64 bits by central differences of step h
    (error of order h^2) at a few places, against the 32-bit kernel's."""
    x, gamma, beta, g = norm_inputs(3, 50, "f32", "f32")
    dy = normal(g, 3, 50)
    _, mean, rstd = zc.layer_norm(x, gamma, beta, stats=True)
    dx, dgamma, dbeta = zc.layer_norm_grad(dy, x, mean, rstd, gamma)

    def f(x, gamma, beta):
        m = x.mean(1, keepdim=True)
        y = (x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + 1e-5) * gamma + beta
        return float((dy.double() * y).sum())

    args = [x.double(), gamma.double(), beta.double()]
    for which, got in ((0, dx), (1, dgamma), (2, dbeta)):
        for i in range(0, got.numel(), 7):
            h, v = 1e-5, []
            for s in (h, -h):
                a = [t.clone() for t in args]
                a[which].view(-1)[i] += s
                v.append(f(*a))
            assert abs((v[0] - v[1]) / (2 * h) - float(got.reshape(-1)[i])) <= 2e-5, (which, i)


def test_layer_norm_no_rows(zc):
    x = torch.empty(0, 64, device="cuda")
    assert zc.layer_norm(x).shape == (0, 64)
    n = torch.empty(0, device="cuda")
    dx, dgamma, dbeta = zc.layer_norm_grad(x, x, n, n)
    assert dx.shape == (0, 64) and not dgamma.any() and not dbeta.any()


# ------------------------------------------------------------- distillation
def teach(g, rows, vocab, top, t, it=torch.int64, ragged=True):
    student = (2.5 * normal(g, rows, vocab)).to(TYPES[t])
    top_ = min(top, vocab)
    teacher = (3 * normal(g, rows, top)).to(TYPES[t])
    index = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:top_] for _ in range(rows)])
    if top_ < top:
        index = torch.cat([index, torch.full((rows, top - top_), -1, device="cuda")], 1)
    if ragged and top > 1:
        index[rows // 2, 1:] = -1
    return student, teacher, index.to(it)


def ref_distill(logits, teacher, index, T, weight, dloss):
    """loss, lse, dlogits in 64 bits, and the error that 32-bit arithmetic may bring to each."""
    z = logits.double() / T
    rows = z.shape[0]
    w = torch.ones(rows, device="cuda").double() if weight is None else weight.double()
    c = T * w * (1.0 if dloss is None else dloss.double())
    lp = torch.log_softmax(torch.where(index >= 0, teacher.double() / T, -math.inf), 1)
    empty = (index < 0).all(1) | ((index < 0) | (teacher == -math.inf)).all(1)
    at = index.clamp(min=0).long()
    p = torch.where(empty[:, None] | (index < 0), 0.0, lp.exp())
    lse = torch.logsumexp(z, 1)
    lq = z.gather(1, at) - lse[:, None]
    loss = torch.where(empty | (w == 0), 0.0, w * T * T * torch.where(p > 0, p * (lp - lq), 0.0).sum(1))
    q = torch.exp(z - lse[:, None])
    d = q.scatter_add(1, at, -p)
    dead = (empty | (c == 0))[:, None]
    d = torch.where(dead, 0.0, c[:, None] * d)
    # An argument of exp() is off by a few roundings of z and lse, whose size is bounded by big; the sums are in chains
    # of at most vocab / 256 + 16 <= 600 positive terms, an error that the logarithm passes on as it is.
    fin = z.masked_fill(~z.isfinite(), 0.0).abs().amax(1) + lse.abs().nan_to_num(0, 0, 0)
    tfin = (teacher.double() / T).masked_fill(~teacher.isfinite(), 0.0).abs().amax(1) if teacher.shape[1] else 0.0 * fin
    chain = min(z.shape[1], 600) + 16
    e = (4 * E * (fin + tfin + 4) + chain * E)
    size = torch.where(p > 0, p * (lp.abs() + z.gather(1, at).abs()), 0.0).sum(1) + lse.abs()
    tl = w.abs() * T * T * (e * (1 + size) + 8 * E * size)
    td = c.abs()[:, None] * e[:, None] * 2 * (q + torch.zeros_like(q).scatter_add(1, at, p))
    return loss, torch.where(empty | (w == 0), 0.0, lse), d, tl, e * (1 + 0 * lse), td


def check_distill(zc, student, teacher, index, T, weight, dloss):
    loss, lse, d, tl, te, td = ref_distill(student, teacher, index, T, weight, dloss)
    kw = {"temperature": T, "weight": weight}
    got_loss, got_lse = zc.distill_loss(student, teacher, index, **kw)
    within(got_loss, loss, tl + E * loss.abs(), "loss")
    within(got_lse, lse, te + 2 * E * lse.abs(), "lse")
    tol = td + U[student.dtype] * (d.abs() + td) + S[student.dtype]
    got = zc.distill_grad(student, teacher, index, got_lse, dloss, **kw)
    within(got, d, tol, "grad")
    both_loss, both = zc.distill_value_and_grad(student, teacher, index, dloss, **kw)
    within(both_loss, loss, tl + E * loss.abs(), "loss of both")
    within(both, d, tol, "grad of both")
    return both_loss, both


DISTILL_SIZES = [(1, 1, 1), (2, 3, 5), (3, 17, 4), (5, 64, 1), (4, 257, 64), (7, 1000, 17), (2, 4096, 64), (3, 5003, 100),
                 (2, 32003, 20), (1, 50001, 256), (2, 70001, 1024), (1, 131072, 64), (2, 131071, 33), (150, 2048, 8)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,vocab,top", DISTILL_SIZES)
def test_distill(zc, rows, vocab, top, t):
    g = gen(2)
    student, teacher, index = teach(g, rows, vocab, top, t, torch.int32 if vocab % 2 else torch.int64)
    weight = torch.rand(rows, generator=g, device="cuda") + 0.1
    dloss = normal(g, rows)
    check_distill(zc, student, teacher, index, 2.0, weight, dloss)
    check_distill(zc, student, teacher, index, 0.7, None, None)


@pytest.mark.parametrize("t,rows,vocab", [("f32", 2, 450001), ("bf16", 1, 900003), ("f16", 3, 262145), ("f32", 3, 131073),
                                          ("bf16", 700, 513), ("f16", 1200, 100), ("f32", 400, 9001)])
def test_distill_by_the_size_of_a_row(zc, rows, vocab, t):
    """Rows in one block, in clusters of each size, and beyond what a cluster holds."""
    g = gen(21)
    student, teacher, index = teach(g, rows, vocab, 12, t)
    check_distill(zc, strided(student, 1, 0), teacher, index, 2.0, None, torch.rand(rows, generator=g, device="cuda"))


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("pitch,shift", [(1, 0), (8, 8), (5, 3)])
@pytest.mark.parametrize("vocab", [1001, 4096, 40007])
def test_distill_strides_and_in_place(zc, vocab, pitch, shift, t):
    g = gen(3)
    student, teacher, index = teach(g, 6, vocab, 9, t)
    wide = strided(student, pitch, shift)
    teacher2, index2 = strided(teacher, 2, 1), strided(index, 3, 1)
    check_distill(zc, wide, teacher2, index2, 1.5, None, None)
    kw = {"temperature": 1.5}
    loss, d = zc.distill_value_and_grad(student, teacher, index, **kw)
    loss2, d2 = zc.distill_value_and_grad(wide, teacher2, index2, **kw)
    tol = 1e-5 * d.double().abs().amax() + U[student.dtype] * 2 * d.double().abs() + S[student.dtype]
    within(d2, d.double(), tol)
    _, lse = zc.distill_loss(student, teacher, index, **kw)
    want = zc.distill_grad(student, teacher, index, lse, **kw)
    a, b = student.clone(), student.clone()
    assert torch.equal(zc.distill_value_and_grad(a, teacher, index, out=a, **kw)[1], d) and torch.equal(a, d)
    assert torch.equal(zc.distill_grad(b, teacher, index, lse, out=b, **kw), want) and torch.equal(b, want)


@pytest.mark.parametrize("vocab", [300, 33000])
def test_distill_rows_that_are_masked(zc, vocab):
    """Padding rows hold anything, NaN included, and give exact zeros; their neighbours are untouched."""
    g = gen(4)
    student, teacher, index = teach(g, 8, vocab, 6, "f32", ragged=False)
    want_loss, want = zc.distill_value_and_grad(student, teacher, index, temperature=2.0)
    weight, dloss = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    student[1], weight[1] = float("nan"), 0.0
    index[3] = -1
    student[3] = float("inf")
    teacher[5] = -math.inf
    student[5] = float("nan")
    kw = {"temperature": 2.0, "weight": weight}
    loss, d = zc.distill_value_and_grad(student, teacher, index, dloss, **kw)
    loss2, lse = zc.distill_loss(student, teacher, index, **kw)
    d2 = zc.distill_grad(student, teacher, index, lse, dloss, **kw)
    dead = torch.tensor([1, 3, 5], device="cuda")
    live = torch.tensor([0, 2, 4, 6, 7], device="cuda")
    for t in (loss, loss2, lse, d, d2):
        assert not t[dead].any()
    assert torch.equal(loss[live], want_loss[live]) and torch.equal(d[live], want[live])
    within(d2[live], want[live].double(), 1e-6 * want.double().abs().amax())
    dloss[2] = 0.0
    loss3, d3 = zc.distill_value_and_grad(student, teacher, index, dloss, **kw)
    assert torch.equal(loss3, loss) and not d3[2].any() and not zc.distill_grad(student, teacher, index, lse, dloss, **kw)[2].any()


@pytest.mark.parametrize("vocab", [200, 40000])
def test_distill_infinities_and_repeats(zc, vocab):
    g = gen(5)
    student, teacher, index = teach(g, 5, vocab, 6, "f32", ragged=False)
    student[0, :vocab // 2] = -math.inf  # forbidden tokens, the teacher's among the others
    index[0] = torch.arange(vocab - 6, vocab, device="cuda")
    teacher[1, 2] = -math.inf  # an entry without weight, at a token that the student forbids
    student[1, index[1, 2]] = -math.inf
    student[2].fill_(torch.finfo(torch.float32).min)  # a mask of the type's lowest value
    student[2, index[2]] = 1.0
    index[3] = index[3, 0]  # one token six times
    index[4, 3:] = index[4, :3].flip(0)
    check_distill(zc, student, teacher, index, 1.3, None, None)
    student[1, index[1, 0]] = -math.inf  # now the teacher wants a forbidden token
    loss, d = zc.distill_value_and_grad(student, teacher, index, temperature=1.3)
    assert float(loss[1]) == math.inf and bool(d[1].isfinite().all()) and float(d[1, index[1, 0]]) < 0


def test_distill_bad_index_poisons_its_row_only(zc):
    g = gen(6)
    student, teacher, index = teach(g, 4, 500, 5, "f16", ragged=False)
    loss, d = zc.distill_value_and_grad(student, teacher, index)
    _, lse = zc.distill_loss(student, teacher, index)
    for bad in (500, -2, 1 << 40):
        i = index.clone()
        i[2, 3] = bad
        loss2, d2 = zc.distill_value_and_grad(student, teacher, i)
        d3 = zc.distill_grad(student, teacher, i, lse)
        assert bool(loss2[2].isnan()) and bool(d2[2].isnan().all()) and bool(d3[2].isnan().all())
        keep = torch.tensor([0, 1, 3], device="cuda")
        assert torch.equal(loss2[keep], loss[keep]) and torch.equal(d2[keep], d[keep])


def test_distill_gradient_against_differences(zc):
    g = gen(7)
    student, teacher, index = teach(g, 3, 40, 6, "f32")
    dloss = normal(g, 3)
    _, d = zc.distill_value_and_grad(student, teacher, index, dloss, temperature=1.7)

    def f(s):
        return float((dloss.double() * ref_distill(s, teacher, index, 1.7, None, None)[0]).sum())

    h = 1e-4
    for i in range(0, 120, 7):
        v = []
        for s in (h, -h):
            a = student.double().clone()
            a.view(-1)[i] += s
            v.append(f(a))
        assert abs((v[0] - v[1]) / (2 * h) - float(d.view(-1)[i])) <= 1e-5, i


def test_distill_no_rows_and_no_entries(zc):
    x = torch.empty(0, 9, device="cuda")
    loss, d = zc.distill_value_and_grad(x, torch.empty(0, 2, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"))
    assert loss.shape == (0,) and d.shape == (0, 9)
    x = torch.ones(3, 9, device="cuda")
    loss, d = zc.distill_value_and_grad(x, torch.empty(3, 0, device="cuda"), torch.empty(3, 0, dtype=torch.int64, device="cuda"))
    assert not loss.any() and not d.any()


# ------------------------------------------------------------- 8-bit integers
def ref_quantize(x):
    """In 32 bits on the CPU: the definition is of 32-bit numbers, and its division and rounding are exact there."""
    x = x.float().cpu()
    if x.shape[1] == 0:
        return torch.zeros(x.shape, dtype=torch.int8), torch.zeros(x.shape[0])
    m = x.abs().amax(1)
    scale = torch.where(m.isfinite(), m / 127, float("nan"))
    q = torch.round(x / scale[:, None]).clamp(-127, 127)
    q = torch.where((scale > 0)[:, None], q, 0.0)
    return q.to(torch.int8), scale


def ref_product(q, s, w, sw, bias):
    y = (q.double().cpu() @ w.double().cpu().t()) * s.double().cpu()[:, None] * sw.double().cpu()
    return y, (y if bias is None else y + bias.double().cpu())


def check_product(got, q, s, w, sw, bias):
    y, want = ref_product(q, s, w, sw, bias)
    t32 = 4 * E * (y.abs() + want.abs())  # the sum's conversion, two scales, the bias
    within(got.cpu(), want, t32 + U[got.dtype] * (want.abs() + t32) + S[got.dtype], "product")


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (2, 16), (7, 33), (5, 784), (3, 1001), (4, 4096), (2, 8197), (2, 40000)])
def test_quantize(zc, rows, cols, t):
    g = gen(8)
    x = (normal(g, rows, cols) * torch.exp(normal(g, rows, 1))).to(TYPES[t])
    for v in (x, strided(x, 3, 1), strided(x, 16, 8)):
        q, s = zc.quantize_rows(v)
        wq, ws = ref_quantize(v)
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


def test_quantize_rows_out_of_the_ordinary(zc):
    x = torch.ones(6, 100, device="cuda")
    x[0] = 0.0
    x[1, 3] = float("nan")
    x[2, 99] = float("-inf")
    x[3] = 1e-44  # the scale underflows
    x[4, 1:] = -3e38
    x[5] = torch.arange(100, device="cuda") - 49.5
    q, s = zc.quantize_rows(x)
    wq, ws = ref_quantize(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu().nan_to_num(-1), ws.nan_to_num(-1))
    assert bool(s[1].isnan()) and bool(s[2].isnan()) and not q[:3].any()


MUL_SIZES = [(1, 1, 1), (1, 5, 3), (2, 16, 64), (3, 100, 33), (1, 1000, 784), (1, 4096, 1024), (4, 257, 4096), (8, 512, 513),
             (15, 300, 1001), (16, 128, 128), (17, 256, 256), (31, 1000, 130), (33, 64, 2048), (64, 384, 784), (65, 129, 300),
             (100, 1024, 512), (128, 128, 4096), (129, 257, 1025), (200, 4099, 1001), (256, 512, 16), (300, 700, 15),
             (512, 512, 512), (1000, 130, 777), (3, 40, 20000), (130, 260, 8200)]


def ints(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,n,k", MUL_SIZES)
def test_int8_matmul(zc, m, n, k, t):
    g = gen(9)
    a, b = ints(g, m, k), ints(g, n, k)
    sa, sb = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda") / k
    bias = normal(g, n)
    pad = (k + 15) // 16 * 16 - k
    for x, w in ((a, b), (strided(a, pad), strided(b, pad)), (strided(a, pad + 16, 16), strided(b, 1, 0)), (strided(a, 5, 3), b)):
        for bi in (None, bias):
            check_product(zc.int8_matmul(x, sa, w, sb, bi, dtype=TYPES[t]), a, sa, b, sb, bi)
    out = strided(torch.zeros(m, n, device="cuda", dtype=TYPES[t]), 3, 1)
    got = zc.int8_matmul(strided(a, pad), sa, strided(b, pad), sb, bias, out=out)
    check_product(got, a, sa, b, sb, bias)
    wide = out._base
    assert bool(wide[:, 0].isnan().all()) and bool(wide[:, n + 1:].isnan().all())  # nothing beside it is written


@pytest.mark.parametrize("rows", [1, 3, 40])
def test_int8_sums_to_the_last_bit(zc, rows):
    """The longest inner axis, every product at its largest: the sum is exact up to 2^31 - 16384."""
    k = 131071
    a = torch.full((rows, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((5, k), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    b[2, ::2] = 127
    b[3] = 1
    one = torch.ones(rows, device="cuda")
    for x, w in ((a, b), (strided(a, 1), strided(b, 1))):
        got = zc.int8_matmul(x, one, w, torch.ones(5, device="cuda"))
        want = (a[:1].cpu().long() * b.cpu().long()).sum(1)
        assert torch.equal(got.cpu(), want.float().expand(rows, 5)), (got[0], want)


def test_int8_empty_products(zc):
    g = gen(10)
    one = torch.ones(4, device="cuda")
    assert zc.int8_matmul(ints(g, 0, 7), one[:0], ints(g, 4, 7), one).shape == (0, 4)
    assert zc.int8_matmul(ints(g, 4, 7), one, ints(g, 0, 7), one[:0]).shape == (4, 0)
    y = zc.int8_matmul(ints(g, 4, 0), one, ints(g, 4, 0), one, bias=2 * one)
    assert torch.equal(y, torch.full((4, 4), 2.0, device="cuda"))


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 1000, 784), (1, 4096, 1024), (2, 513, 4096), (5, 300, 1001), (9, 256, 255),
                                   (16, 512, 512), (40, 129, 1000), (333, 500, 1001), (512, 1024, 784)])
def test_int8_linear(zc, m, n, k, t):
    g = gen(11)
    x = (normal(g, m, k) * torch.exp(normal(g, m, 1))).to(TYPES[t])
    layer = zc.Int8Linear.from_float(normal(g, n, k), normal(g, n))
    plain = zc.Int8Linear(layer.weight.contiguous(), layer.scale)
    q, s = ref_quantize(x)
    for v in (x, strided(x, 5, 3), strided(x, 8, 8)):
        check_product(layer(v), q, s, layer.weight, layer.scale, layer.bias)
        check_product(plain(v), q, s, layer.weight, layer.scale, None)
    # the same as the two calls that it stands for
    a, sa = zc.quantize_rows(x)
    assert torch.equal(layer(x), zc.int8_matmul(a, sa, layer.weight, layer.scale, layer.bias, dtype=x.dtype))


def test_int8_linear_bad_rows_stay_alone(zc):
    g = gen(12)
    for m in (1, 4, 200):
        x = normal(g, m, 500)
        layer = zc.Int8Linear.from_float(normal(g, 300, 500))
        want = layer(x)
        x[m // 2, 7] = float("nan")
        got = layer(x)
        assert bool(got[m // 2].isnan().all())
        keep = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(got[keep], want[keep])
        x[m // 2] = 0.0
        assert not layer(x)[m // 2].any()


# ------------------------------------------------------------- sampling
def ref_sample(x, u, t, k, p, mp, token, slack=1e-6):
    """Whether `token` is the choice in 64 bits, give or take `slack` of the row's weight at each edge, and the log
    probability that it then has: weights from 32-bit exp() are off by less than 2^-22, and a whole-number sum of them by
    less than that of itself."""
    x = x.double()
    V = x.shape[0]
    ok = x.isnan().logical_not() & (x > -math.inf)
    if not bool(ok.any()):
        assert token == -1
        return -math.inf
    x = torch.where(ok, x, torch.tensor(-math.inf, dtype=torch.float64))
    order = torch.sort(x, descending=True, stable=True).indices
    if not t > 0:
        assert token == int(order[0])
        return 0.0
    m = x.amax()
    d = torch.where(x == m, 0.0, (x - m) / t)
    w = torch.where(ok, torch.exp(d), 0.0)
    w = torch.where(w < 2.0 ** -40, 0.0, w)
    rank = torch.empty(V, dtype=torch.long)
    rank[order] = torch.arange(V)
    base = w * (rank < k) if 0 < k < V else w
    ws = base[order]
    before = torch.empty_like(ws)
    before[order] = ws.cumsum(0) - ws
    total = float(ws.sum())
    lo = hi = base  # at least / at most kept
    if p < 1:
        pp = max(p, 0.0)
        lo = base * ((before < (pp - slack) * total) | (rank == 0))
        hi = base * ((before < (pp + slack) * total) | (rank == 0))
    if mp > 0:
        e = min(mp, 1.0)
        lo = lo * ((w >= e * (1 + slack)) | (w == 1))
        hi = hi * ((w >= e * (1 - slack)) | (w == 1))
    assert float(hi[token]) > 0, "token %d is not kept" % token
    first, last = float(lo[:token].sum()), float(hi[:token + 1].sum())
    least, most = float(lo.sum()), float(hi.sum())
    eps = slack * total
    assert first - eps <= u * most and u * least <= last + eps, (token, first, last, u, least, most)
    return float(d[token]) - math.log(0.5 * (least + most)), max(1e-5, 2 * (most - least) / least) + 4 * E * abs(float(d[token]))


def check_sample(zc, logits, u, t, k, p, mp):
    token, logprob = zc.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp)
    xs, us, tok, lp = logits.float().cpu(), u.double().cpu(), token.tolist(), logprob.double().tolist()
    rows = xs.shape[0]
    at = lambda v, i, d: d if v is None else float(v[i])
    for i in range(rows):
        r = ref_sample(xs[i], float(us[i]), at(t, i, 1.0), int(at(k, i, 0)), at(p, i, 1.0), at(mp, i, 0.0), tok[i])
        if isinstance(r, tuple):
            assert abs(lp[i] - r[0]) <= r[1], (i, lp[i], r)
        else:
            assert lp[i] == r, (i, lp[i], r)
    return token, logprob


def rules(g, rows):
    r = torch.rand(rows, 4, generator=g, device="cuda")
    t = torch.where(r[:, 0] < 0.1, 0.0, 0.3 + 2 * torch.rand(rows, generator=g, device="cuda"))
    k = torch.where(r[:, 1] < 0.5, torch.randint(1, 300, (rows,), generator=g, device="cuda"), 0).to(torch.int32)
    p = torch.where(r[:, 2] < 0.6, torch.rand(rows, generator=g, device="cuda"), 1.0)
    mp = torch.where(r[:, 3] < 0.3, 0.2 * torch.rand(rows, generator=g, device="cuda"), 0.0)
    return t, k, p, mp


VOCABS = [1, 2, 5, 31, 33, 100, 1000, 1023, 1025, 2049, 5003, 8192, 32003, 50001, 131071, 131072, 262147]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("vocab", VOCABS)
def test_sample(zc, vocab, t):
    g = gen(13)
    rows = 24 if vocab < 40000 else 8
    x = 2.5 * normal(g, rows, vocab)
    x[:, :max(1, vocab // 100)] += 5
    x = x[:, torch.randperm(vocab, generator=g, device="cuda")].to(TYPES[t])
    x[torch.rand(rows, vocab, generator=g, device="cuda") < 0.02] = -math.inf
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64 if vocab % 2 else torch.float32)
    r = rules(g, rows)
    token, logprob = check_sample(zc, x, u, *r)
    check_sample(zc, x, u, r[0], None, None, None)
    check_sample(zc, x, u, None, r[1], None, None)
    check_sample(zc, x, u, None, None, r[2], None)
    check_sample(zc, x, u, None, None, None, r[3])
    # a row's token does not depend on the rows beside it or on where the row lies
    for i in range(0, rows, 5):
        one = zc.sample(strided(x[i:i + 1], 3, 1), u[i:i + 1], *[v[i:i + 1] for v in r])
        assert int(one[0]) == int(token[i]) and float(one[1]) == float(logprob[i])
    many = zc.sample(x.repeat(40, 1), u.repeat(40), *[v.repeat(40) for v in r])
    assert torch.equal(many[0], token.repeat(40)) and torch.equal(many[1], logprob.repeat(40))


@pytest.mark.parametrize("vocab", [7, 3000, 70000])
def test_sample_equal_logits(zc, vocab):
    """All weights are equal, so every edge is exact: ranks are by index, and so is the choice."""
    rows = 64
    x = torch.zeros(rows, vocab, device="cuda")
    x[:, ::2] = -0.0  # equal to 0
    u = (torch.arange(rows, device="cuda", dtype=torch.float64) + 0.5) / rows
    at = (torch.arange(rows, dtype=torch.float64) + 0.5) / rows
    for k in (1, 2, 5, vocab - 1, vocab, vocab + 1, 0, -3):
        n = k if 0 < k < vocab else vocab
        token, logprob = zc.sample(x, u, top_k=k)
        assert torch.equal(token.cpu(), (at * n).long())
        assert abs(float(logprob[0]) + math.log(n)) <= 1e-6 * (1 + math.log(n))
        for p in (0.0, 0.25, 0.5, 1.0):
            kept = n if p >= 1 else max(1, math.ceil(p * n))  # these p times n are exact in 64 bits
            for mp in (0.0, 0.3, 1.0, 2.0):
                token, _ = zc.sample(x, u, top_k=k, top_p=p, min_p=mp)
                assert torch.equal(token.cpu(), (at * kept).long()), (k, p, mp)
    for T in (1e-3, 1e30, math.inf):
        assert torch.equal(zc.sample(x, u, temperature=T)[0].cpu(), (at * vocab).long())


def test_sample_frequencies(zc):
    """With uniforms on an even grid of n, a token of probability p is drawn n p times, give or take one for the grid's
    ends and the weights' error."""
    g = gen(14)
    n, vocab = 4096, 500
    x = (2 * normal(g, 1, vocab)).expand(n, vocab).contiguous()
    u = (torch.arange(n, device="cuda", dtype=torch.float64) + 0.5) / n
    count = torch.bincount(zc.sample(x, u, temperature=1.5)[0], minlength=vocab).double()
    want = n * torch.softmax(x[0].double() / 1.5, 0)
    assert float((count - want).abs().amax()) <= 1.0 + 1e-3


@pytest.mark.parametrize("vocab", [60, 40000])
def test_sample_rows_out_of_the_ordinary(zc, vocab):
    g = gen(15)
    x = normal(g, 12, vocab)
    x[0] = -math.inf
    x[1] = float("nan")
    x[2] = -math.inf
    x[2, vocab // 3] = -5.0  # one token is left
    x[3, 5] = x[3, 20] = math.inf  # only these two have weight
    x[4, ::3] = float("nan")
    x[5] = torch.finfo(torch.float32).min  # masked with the lowest value: all alike
    x[6, 11] = torch.finfo(torch.float32).max
    x[7, 9] = 40.0  # far above the rest
    for u in (0.0, 0.4, 0.9999999, 1.0, 5.0, -1.0, float("nan")):
        us = torch.full((12,), u, device="cuda")
        for kw in ({}, {"top_k": 1}, {"top_k": 3, "top_p": 0.8}, {"top_p": 0.3}, {"min_p": 0.5}, {"temperature": 0.0},
                   {"temperature": -1.0}, {"temperature": float("nan")}, {"top_p": float("nan")}, {"min_p": float("nan")}):
            token, logprob = zc.sample(x, us, **kw)
            tok = token.tolist()
            assert tok[0] == tok[1] == -1 and tok[2] == vocab // 3
            assert logprob[0] == logprob[1] == -math.inf and logprob[2] == 0
            assert tok[3] in (5, 20) and (u < 0.5 or not 0.5 <= u or kw or tok[3] == 20)
            assert tok[4] % 3 and 0 <= tok[4] < vocab and tok[6] == 11 and tok[7] == 9
            assert 0 <= min(tok[2:]) and max(tok) < vocab
            if u == 0.0 and "top_k" not in kw and kw.get("temperature", 1.0) > 0 and kw.get("top_p", 1.0) != 0.3 and "min_p" not in kw:
                assert tok[8] == 0  # the first index
            if not kw.get("temperature", 1.0) > 0 or kw.get("top_k") == 1:
                assert tok[8:] == x[8:].argmax(1).tolist() and tok[5] == 0


def test_sample_wide_temperatures(zc):
    g = gen(16)
    x = 3 * normal(g, 16, 20000)
    u = torch.rand(16, generator=g, device="cuda")
    for T in (1e-30, 1e-3, 0.05, 5.0, 100.0, 1e6):
        t = torch.full((16,), T, device="cuda")
        for k, p in ((0, 1.0), (40, 1.0), (0, 0.5), (5000, 0.9)):
            check_sample(zc, x, u, t, torch.full((16,), k, dtype=torch.int32, device="cuda"), torch.full((16,), p, device="cuda"), None)


def test_sample_no_rows(zc):
    token, logprob = zc.sample(torch.empty(0, 9, device="cuda"), torch.empty(0, device="cuda"))
    assert token.shape == logprob.shape == (0,)


# ------------------------------------------------------------- all of them
def test_results_do_not_depend_on_the_run(zc):
    g = gen(17)
    x, gamma, beta, _ = norm_inputs(501, 1003, "bf16", "f32")
    dy = (0.01 * normal(g, 501, 1003)).to(torch.bfloat16)
    _, mean, rstd = zc.layer_norm(x, gamma, beta, stats=True)
    student, teacher, index = teach(g, 9, 60001, 50, "bf16")
    layer = zc.Int8Linear.from_float(normal(g, 700, 1003))
    logits = (3 * normal(g, 9, 60001)).to(torch.bfloat16)
    u = torch.rand(9, generator=g, device="cuda")
    run = lambda: (*zc.layer_norm_grad(dy, x, mean, rstd, gamma), *zc.distill_value_and_grad(student, teacher, index),
                   layer(x), *zc.sample(logits, u, top_k=500, top_p=0.9))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), first))


def test_other_streams(zc):
    """A call on a stream of its own waits for nothing on the current one, and its results belong to it."""
    g = gen(18)
    x, gamma, beta, _ = norm_inputs(40, 1024, "bf16", "f32")
    student, teacher, index = teach(g, 9, 5000, 20, "bf16")
    layer = zc.Int8Linear.from_float(normal(g, 700, 1024))
    u = torch.rand(9, generator=g, device="cuda")
    _, mean, rstd = zc.layer_norm(x, gamma, beta, stats=True)

    def run(**kw):
        return (zc.layer_norm(x, gamma, beta, **kw), *zc.layer_norm_grad(x, x, mean, rstd, gamma, **kw),
                *zc.distill_value_and_grad(student, teacher, index, **kw), *zc.distill_loss(student, teacher, index, **kw),
                layer(x, **kw), *zc.quantize_rows(x, **kw), *zc.sample(student, u, top_k=50, top_p=0.9, **kw))

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = run(stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(side):
        again = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_in_a_cuda_graph(zc):
    g = gen(19)
    x, gamma, beta, _ = norm_inputs(16, 1024, "bf16", "f32")
    layer = zc.Int8Linear.from_float(normal(g, 5000, 1024))
    u = torch.rand(16, generator=g, device="cuda")
    dy = (0.01 * normal(g, 16, 1024)).to(torch.bfloat16)
    teacher, index = 3 * normal(g, 16, 8), torch.randint(0, 5000, (16, 8), generator=g, device="cuda")

    def step():
        h, mean, rstd = zc.layer_norm(x, gamma, beta, stats=True)
        logits = layer(h)
        token, logprob = zc.sample(logits, u, top_k=40, top_p=0.9)
        loss, d = zc.distill_value_and_grad(logits, teacher, index)
        return (h, logits, token, logprob, loss, d, *zc.layer_norm_grad(dy, x, mean, rstd, gamma))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(normal(g, 16, 1024))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_front_end_refusals(zc):
    x = torch.zeros(4, 8, device="cuda")
    i = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    v = torch.zeros(4, device="cuda")
    q = torch.zeros(4, 8, dtype=torch.int8, device="cuda")
    bad = [
        (lambda: zc.layer_norm(x.double()), "NotSupported"), (lambda: zc.layer_norm(x.t()), "NonContiguous"),
        (lambda: zc.layer_norm(x, v), "ShapeMismatch"), (lambda: zc.layer_norm(x, torch.zeros(8)), "DeviceMismatch"),
        (lambda: zc.layer_norm(x, torch.ones(8, device="cuda"), torch.ones(8, device="cuda").half()), "DTypeMismatch"),
        (lambda: zc.layer_norm(x, out=x.half()), "DTypeMismatch"), (lambda: zc.layer_norm(x[0]), "InvalidShape"),
        (lambda: zc.layer_norm(x[:1].expand(4, 8)), "NonContiguous"), (lambda: zc.layer_norm(x, eps=-1.0), "InvalidArgument"),
        (lambda: zc.layer_norm(x[:, :0]), "InvalidShape"),
        (lambda: zc.layer_norm_grad(x.half(), x, v, v), "DTypeMismatch"), (lambda: zc.layer_norm_grad(x, x, v[:3], v), "ShapeMismatch"),
        (lambda: zc.layer_norm_grad(x[:3], x, v, v), "ShapeMismatch"), (lambda: zc.layer_norm_grad(x, x, v.double(), v), "DTypeMismatch"),
        (lambda: zc.distill_loss(x, x[:, :2], i.short()), "NotSupported"), (lambda: zc.distill_loss(x, x[:, :3], i), "ShapeMismatch"),
        (lambda: zc.distill_loss(x, x[:3, :2], i), "ShapeMismatch"), (lambda: zc.distill_loss(x, x[:, :2], i, temperature=0.0), "InvalidArgument"),
        (lambda: zc.distill_loss(x, x[:, :2], i, weight=v[:2]), "ShapeMismatch"),
        (lambda: zc.distill_grad(x, x[:, :2], i, v.half()), "DTypeMismatch"),
        (lambda: zc.distill_value_and_grad(x, x[:, :2], i, out=x[:3]), "ShapeMismatch"),
        (lambda: zc.quantize_rows(q), "NotSupported"), (lambda: zc.int8_matmul(x, v, q, v), "DTypeMismatch"),
        (lambda: zc.int8_matmul(q, v, q[:, :7], v), "ShapeMismatch"), (lambda: zc.int8_matmul(q, v[:3], q, v), "ShapeMismatch"),
        (lambda: zc.int8_matmul(q, v, q, v, dtype=torch.int32), "NotSupported"),
        (lambda: zc.Int8Linear(x, v), "DTypeMismatch"), (lambda: zc.Int8Linear(q, v)(x[:, :7]), "ShapeMismatch"),
        (lambda: zc.sample(x, v.half()), "NotSupported"), (lambda: zc.sample(x, v[:2]), "ShapeMismatch"),
        (lambda: zc.sample(x, v, top_k=v), "DTypeMismatch"), (lambda: zc.sample(x, v, temperature=v[:1]), "ShapeMismatch"),
    ]
    for n, (f, name) in enumerate(bad):
        with pytest.raises(zc.ZpuCudaError) as e:
            f()
        assert e.value.name == name, (n, e.value)


def test_older_entry_points_refuse_bf16(zc):
    a = torch.zeros(4, 4, dtype=torch.bfloat16, device="cuda")
    for f in (lambda: zc.matmul(a, a), lambda: zc.tensor_copy(a, torch.zeros(4, 4, device="cuda"))):
        with pytest.raises(zc.ZpuCudaError) as e:
            f()
        assert e.value.name == "NotSupported"


def test_example_trains_and_serves(zc):
    """The example's head learns: the loss falls by more than half, and most of its likeliest tokens are among the
    teacher's (a chance of 32 / 1024 before training)."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "lm_head.py")
    spec = importlib.util.spec_from_file_location("lm_head", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    losses, agree, drawn, logprob = module.main(["--tokens", "200", "--width", "128", "--vocab", "1024", "--steps", "40"])
    assert losses[-1] < 0.5 * losses[0] and agree > 0.5
    assert bool(((drawn >= 0) & (drawn < 1024)).all()) and bool((logprob <= 0).all())


def test_example_gradients_against_torch(zc):
    """The example's whole backward pass against autograd of the same head in 64 bits (products by 3xTF32, 1e-5)."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "lm_head.py")
    spec = importlib.util.spec_from_file_location("lm_head", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    g = gen(20)
    head = module.Head(96, 500)
    x = normal(g, 70, 96)
    teacher, index = (3 * normal(g, 70, 500)).topk(10, 1)
    loss, grads = head.value_and_grad(x, teacher, index, 2.0)
    leaves = [t.double().requires_grad_() for t in (x, head.gamma, head.beta, head.weight)]
    h = torch.nn.functional.layer_norm(leaves[0], (96,), leaves[1], leaves[2])
    logq = torch.log_softmax(h @ leaves[3].t() / 2.0, 1).gather(1, index)
    p = torch.softmax(teacher.double() / 2.0, 1)
    want = 4.0 * (p * (p.log() - logq)).sum(1).mean()
    want.backward()
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    for got, leaf in zip(grads, leaves):
        assert float((got.double() - leaf.grad).norm() / leaf.grad.norm()) <= 2e-5


# ------------------------------------------------------------- sizes at which the split of a row changes
def row_splits(piece):
    """Columns about the sizes at which a row gets another number of threads, for pieces of `piece` elements."""
    return [c for n in (32, 64, 128, 256, 512, 1024, 2048, 4096) for c in (n * piece - 1, n * piece, n * piece + 3)]


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_layer_norm_by_the_threads_of_a_row(zc, t):
    for cols in row_splits(4 if t == "f32" else 8):
        for rows, pitch, shift in ((3, 0, 0), (310, 1, 1)):
            if rows * cols > 4 << 20:
                rows = 4
            x, gamma, beta, _ = norm_inputs(rows, cols, t, "f32", seed=cols, pitch=pitch, shift=shift)
            y = check_norm(zc, x, gamma, beta)
            # a row's result depends neither on the rows beside it nor on where it lies
            assert torch.equal(y[2:3], zc.layer_norm(x[2:3].contiguous(), gamma, beta))


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("cols", [255, 256, 257, 511, 512, 513, 1023, 1025, 2047, 2049, 4095, 4097, 8191, 8193, 16385])
def test_layer_norm_grad_by_the_threads_of_a_row(zc, cols, t):
    check_norm_grad(zc, 11, cols, t, "f32", pitch=1, shift=1)
    check_norm_grad(zc, 330 if cols < 5000 else 80, cols, t, "f32")


@pytest.mark.parametrize("t", list(TYPES))
def test_quantize_by_the_threads_of_a_row(zc, t):
    g = gen(21)
    for cols in row_splits(4 if t == "f32" else 8):
        x = (normal(g, 5, cols) * torch.exp(normal(g, 5, 1))).to(TYPES[t])
        # values about halfway between two whole numbers of scales
        x[:, 1:cols // 2] = ((torch.randint(0, 127, (5, cols // 2 - 1), generator=g, device="cuda") + 0.5)
                             * (x.float().abs().amax(1, keepdim=True) / 127)).to(x.dtype)
        x[3, cols - 1] = float("nan")
        x[4, cols // 2] = float("-inf")
        wq, ws = ref_quantize(x)
        for v in (x, strided(x, 16, 8), strided(x, 1, 1)):
            q, s = zc.quantize_rows(v)
            assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu().nan_to_num(-1), ws.nan_to_num(-1))


# ------------------------------------------------------------- sampling: edges in odd places
@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,spread", [(12, 3000, 0.02), (12, 9001, 0.02), (170, 3000, 0.004), (8, 40000, 0.3), (8, 30000, 1.0)])
def test_sample_sets_that_end_about_zero(zc, rows, vocab, spread, t):
    """Sets of ranks that end among many small logits, with and without many larger ones above them."""
    g = gen(22)
    x = (spread * normal(g, rows, vocab)).to(TYPES[t])
    x[:, 7:400:3] += 3.0
    u = torch.rand(rows, generator=g, device="cuda")
    full = lambda v, d=torch.float32: torch.full((rows,), v, dtype=d, device="cuda")
    for k, p in ((1200, 1.0), (0, 0.6), (0, 0.95), (2000, 0.8), (vocab // 2, 1.0), (vocab // 2, 0.97), (vocab - 1, 0.999)):
        token, logprob = check_sample(zc, x[:12], u[:12], None, full(k, torch.int32)[:12], full(p)[:12], None)
        many = zc.sample(x, u, top_k=full(k, torch.int32), top_p=full(p))  # more rows: other threads a row
        assert torch.equal(many[0][:12], token) and torch.equal(many[1][:12], logprob)


@pytest.mark.parametrize("t", list(TYPES))
def test_sample_ranges_wider_than_a_table(zc, t):
    """Temperatures at which every value from the largest finite one down has weight, and logits out to both its ends."""
    g = gen(23)
    x = normal(g, 10, 20000).to(TYPES[t])
    big = torch.finfo(TYPES[t]).max
    x[:, ::7] *= 100.0
    x[1, 5], x[1, 6], x[2, 9] = big, -big, -big
    x[3] = x[3].abs() * 1e-3
    x[4] = -x[4].abs() - 1.0
    x[5, 30:40] = -math.inf
    x[6, 50:60] = float("nan")
    u = torch.rand(10, generator=g, device="cuda")
    for T in (0.01, 30.0, 1e4, 3e37):
        temp = torch.full((10,), T, device="cuda")
        for k, p in ((0, 1.0), (900, 1.0), (0, 0.7), (15000, 0.9)):
            check_sample(zc, x, u, temp, torch.full((10,), k, dtype=torch.int32, device="cuda"), torch.full((10,), p, device="cuda"), None)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("vocab", [1, 3, 9, 300, 5001])
def test_sample_the_first_of_the_largest(zc, vocab, t):
    """The likeliest token at every place of short rows and the ends of long ones, at every alignment, with equals after it."""
    g = gen(24)
    for shift in range(9):
        places = sorted({c for c in (0, 1, 2, 3, 6, 7, 8, 9, vocab // 2, vocab - 9, vocab - 2, vocab - 1) if 0 <= c < vocab})
        x = strided(normal(g, len(places), vocab).to(TYPES[t]), 2, shift)
        for i, c in enumerate(places):
            x[i, c] = 50.0
            x[i, c + 1::5] = 50.0
        u = torch.rand(len(places), generator=g, device="cuda")
        for kw in ({"temperature": 0.0}, {"top_k": 1}, {"top_p": 0.0}, {"top_k": 450, "top_p": 1e-6}):
            assert zc.sample(x, u, **kw)[0].tolist() == places, (shift, kw)


@pytest.mark.parametrize("t", list(TYPES))
def test_sample_infinite_logits_in_large_sets(zc, t):
    """Infinite logits alone have weight, whatever the set."""
    g = gen(25)
    x = normal(g, 4, 12000).to(TYPES[t])
    x[:, 700] = x[:, 11000] = math.inf
    for kw in ({}, {"top_k": 2000}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_k": 2000, "top_p": 0.999}):
        for u, want in ((0.3, 700), (0.7, 11000)):
            token, logprob = zc.sample(x, torch.full((4,), u, device="cuda"), **kw)
            assert token.tolist() == [want] * 4
            assert float((logprob + math.log(2)).abs().amax()) < 1e-6


def test_sample_refuses_long_rows(zc):
    x = torch.zeros(1, 1 << 22, device="cuda", dtype=torch.float16)
    with pytest.raises(zc.ZpuCudaError) as e:
        zc.sample(x, torch.zeros(1, device="cuda"))
    assert e.value.name == "NotSupported"
    token, logprob = zc.sample(x[:, 1:], torch.full((1,), 0.5, device="cuda", dtype=torch.float64), top_k=1 << 20)
    assert int(token) == 1 << 19 and abs(float(logprob) + 20 * math.log(2)) < 1e-5


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_sample_tiny_temperatures_and_logits(zc, t):
    """Logits and temperatures at the small end of their type: the same tokens as those of both scaled up."""
    g = gen(26)
    x = normal(g, 8, 3000).to(TYPES[t])
    u = torch.rand(8, generator=g, device="cuda")
    for scale in (2.0 ** -40, 2.0 ** -100, 2.0 ** -117):
        for kw in ({}, {"top_p": 0.9}, {"top_k": 1000}, {"top_k": 1000, "top_p": 0.8}):
            want = zc.sample(x, u, temperature=1.0, **kw)
            got = zc.sample((x.double() * scale).to(TYPES[t]), u, temperature=scale, **kw)
            assert torch.equal(got[0], want[0]) and float((got[1] - want[1]).abs().amax()) <= 1e-4


# ------------------------------------------------------------- rows shorter than 16 bytes
SHORT = [("f32", 1, 1), ("f32", 2, 1), ("f32", 1, 2), ("f16", 1, 1), ("f16", 2, 3), ("f16", 6, 1), ("bf16", 1, 6), ("bf16", 3, 2)]


@pytest.mark.parametrize("t,cols,shift", SHORT)
def test_layer_norm_of_rows_inside_16_bytes(zc, t, cols, shift):
    """A first row that begins off the 16-byte grid and ends in the same 16 bytes: nothing that an earlier call left in
    shared memory (here NaN) is among its sums."""
    g = gen(27)
    mess = strided(torch.full((60000, 100), float("nan"), device="cuda", dtype=TYPES[t]), 1, 1)
    ones = torch.ones(60000, device="cuda")
    for rows in (1, 5, 700):
        x, gamma, beta, _ = norm_inputs(rows, cols, t, "f32", seed=cols, pitch=8, shift=shift)
        dy = strided(normal(g, rows, cols).to(TYPES[t]), 8, shift)
        want = zc.layer_norm(x.contiguous(), gamma, beta, stats=True)
        dwant = zc.layer_norm_grad(dy.contiguous(), x.contiguous(), *want[1:], gamma)
        zc.layer_norm(mess)
        assert all(torch.equal(a, b) for a, b in zip(zc.layer_norm(x, gamma, beta, stats=True), want))
        zc.layer_norm_grad(mess, mess, ones, ones)
        assert all(torch.equal(a, b) for a, b in zip(zc.layer_norm_grad(dy, x, *want[1:], gamma), dwant))


# ------------------------------------------------------------- one and two tokens: units of several rows, several rounds
def check_tokens(zc, m, n, k, t):
    """Sums of the 8-bit product of m tokens with n channels, to the last bit, and the whole layer."""
    g = gen(28)
    a, b = ints(g, m, k), ints(g, n, k)
    pad = (k + 15) // 16 * 16 - k
    one = torch.ones(max(m, n), device="cuda")
    want = (a.double() @ b.double().t()).float()  # whole numbers, rounded once
    assert torch.equal(zc.int8_matmul(a, one[:m], strided(b, pad), one[:n]), want)
    layer = zc.Int8Linear(b, torch.rand(n, generator=g, device="cuda") / k, normal(g, n))
    x = (normal(g, m, k) * torch.exp(normal(g, m, 1))).to(TYPES[t])
    q, s = ref_quantize(x)
    for v in (x, strided(x, 3, 1)):
        check_product(layer(v), q, s, b, layer.scale, layer.bias)


@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k", [(5000, 33), (5000, 100), (16384, 500), (16384, 656), (32000, 784), (32000, 816), (16384, 1001),
                                 (5000, 1424), (5120, 1536), (4737, 2000), (8192, 2048), (16384, 2047), (80001, 16), (80001, 333),
                                 (80001, 2048), (50257, 768), (76800, 5000)])
def test_int8_tokens_by_several_rows(zc, m, n, k):
    check_tokens(zc, m, n, k, ("f32", "f16", "bf16")[(n + k) % 3])


# ------------------------------------------------------------- rows over a cluster
@pytest.mark.parametrize("cols", [8193, 16400, 24576, 32769, 40960, 49000, 57344, 65535, 65536])
def test_layer_norm_grad_over_clusters_from_the_first_row_on(zc, cols):
    """Clusters of two to eight blocks whose first exchange is their first or only one: alone, as many as run at a time and
    more, called in a row, with the same bits each time."""
    for rows in (1, 2, 75, 160):
        x, gamma, _, g = norm_inputs(rows, cols, "bf16", "f32", seed=cols)
        dy = (0.01 * normal(g, rows, cols)).to(x.dtype)
        _, mean, rstd = zc.layer_norm(x, gamma, stats=True)
        got = [zc.layer_norm_grad(dy, x, mean, rstd, gamma) for _ in range(8)]
        assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(other, got[0]))
        # a row's dx does not depend on the rows beside it
        one = zc.layer_norm_grad(dy[rows - 1:], x[rows - 1:], mean[rows - 1:], rstd[rows - 1:], gamma)[0]
        assert torch.equal(one[0], got[0][0][rows - 1])
    check_norm_grad(zc, 20, cols, "f32", "f32")


# ------------------------------------------------------------- waits of the 8-bit product that run out
def run_out(zc, m, n, k, t, spin):
    """The product with `spin` tries for its sums: (result, error word, the usual product)."""
    g = gen(29)
    pad = (k + 15) // 16 * 16 - k
    a, b = strided(ints(g, m, k), pad), strided(ints(g, n, k), pad)
    sa, sb, bias = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda") / k, normal(g, n)
    want = zc.int8_matmul(a, sa, b, sb, bias, dtype=TYPES[t])
    out = torch.full((m, n), 7.0, device="cuda", dtype=TYPES[t])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    code = {"f32": 1, "f16": 2, "bf16": 9}[t]
    zc.check(zc.lib().zpucuda_debug_int8_matmul(a.data_ptr(), k + pad, sa.data_ptr(), b.data_ptr(), k + pad, sb.data_ptr(), bias.data_ptr(),
                                                code, out.data_ptr(), n, m, n, k, spin, err.data_ptr(), zc.stream_of()))
    torch.cuda.synchronize()
    # nothing of it stays: the next products are right, and the library's own error word is not set
    assert torch.equal(zc.int8_matmul(a, sa, b, sb, bias, dtype=TYPES[t]), want)
    zc.check(zc.lib().zpucuda_check_device())
    return out, int(err), want


ONE_TILE = [(1, 16384, 4096, "bf16"), (2, 300, 100, "f32"), (1, 80001, 333, "f16"), (9, 1000, 784, "f32"), (5, 512, 4096, "bf16"),
            (40, 129, 8200, "f32"), (333, 4099, 1001, "f16")]


@pytest.mark.parametrize("m,n,k,t", ONE_TILE)
def test_int8_gives_up_and_returns(zc, m, n, k, t):
    """No try for the sums: the call returns, with its copies landed and its products done, and says so."""
    out, err, want = run_out(zc, m, n, k, t, 0)
    assert err == 1
    out, err, want = run_out(zc, m, n, k, t, 1 << 24)
    assert err == 0 and torch.equal(out, want)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(1100, 5000, 300), (1000, 9000, 130), (64, 80001, 200), (3000, 4100, 1000)])
def test_int8_gives_up_on_many_tiles(zc, m, n, k, t):
    """The same where a block has several tiles: a warp that gives up meets the others at the barriers of the tiles to
    come, whether theirs were in time (a few tries: some warps) or not (none)."""
    for spin in (0, 1, 2, 3):
        out, err, want = run_out(zc, m, n, k, t, spin)
        assert err == 1 or torch.equal(out, want)
        assert err == 1 or spin > 0


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m,n,k", [c[:3] for c in ONE_TILE] + [(1100, 5000, 300), (64, 80001, 200)])
def test_int8_gives_nothing_but_nan_after_a_wait(zc, m, n, k, t):
    """What was not waited for is NaN, not part of a sum."""
    assert bool(run_out(zc, m, n, k, t, 0)[0].isnan().all())
    out, err, want = run_out(zc, m, n, k, t, 1)
    assert bool((out.isnan() | (out == want)).all()) and bool(out.isnan().any()) <= err


# ------------------------------------------------------------- the distillation's wait for a row's other blocks
def loss_run_out(zc, rows, vocab, t, spin):
    """The loss with `spin` tries for the sums of the row's other blocks: (loss, lse, error word), and the usual ones."""
    g = gen(30)
    student, teacher, index = teach(g, rows, vocab, 20, t)
    want = zc.distill_loss(student, teacher, index, temperature=1.5)
    loss, lse = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    code = {"f32": 1, "f16": 2, "bf16": 9}
    zc.check(zc.lib().zpucuda_debug_distill_loss(code[t], student.data_ptr(), vocab, zc.head._code("teacher", teacher), teacher.data_ptr(),
                                                 20, 3 if index.dtype == torch.int64 else 4, index.data_ptr(), 20, None, 1.5,
                                                 loss.data_ptr(), lse.data_ptr(), rows, vocab, 20, spin, err.data_ptr(), zc.stream_of()))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(zc.distill_loss(student, teacher, index, temperature=1.5), want))
    zc.check(zc.lib().zpucuda_check_device())
    return loss, lse, int(err), want


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 5000), (3, 70001), (200, 131072), (2000, 40000)])
def test_distill_gives_up_and_returns(zc, rows, vocab, t):
    """Blocks that do not wait for one another's sums: none ends before the others have written theirs to it, and the loss
    is not a number rather than a part of one."""
    loss, lse, err, want = loss_run_out(zc, rows, vocab, t, 0)
    assert err == 1 and bool(loss.isnan().all())
    loss, lse, err, want = loss_run_out(zc, rows, vocab, t, 1 << 24)
    assert err == 0 and torch.equal(loss, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("rows,vocab", [(1, 5000), (3, 70001), (200, 131072)])
def test_distill_gives_no_lse_after_a_wait(zc, rows, vocab):
    """log sum exp, which the gradient is taken from, is NaN like the loss where some of its parts were not waited for."""
    loss, lse, err, want = loss_run_out(zc, rows, vocab, "bf16", 0)
    assert err == 1 and bool(lse.isnan().all())


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("cols", [1, 2, 3, 5])
def test_layer_norm_of_several_rows_in_16_bytes(zc, cols, t):
    """Short rows at their own pitch from every start: the bytes before the matrix (NaN here) are no part of any row, and
    each row comes out as by itself."""
    g = gen(31)
    for shift in range(8):
        for rows in (1, 2, 9, 5000):
            flat = torch.full((shift + rows * cols + 8,), float("nan"), device="cuda", dtype=TYPES[t])
            x = flat[shift:shift + rows * cols].view(rows, cols)
            x.copy_(normal(g, rows, cols))
            dy = torch.full_like(flat, float("nan"))[shift:shift + rows * cols].view(rows, cols)
            dy.copy_(normal(g, rows, cols))
            wide, dwide = strided(x.clone(), 16 - cols), strided(dy.clone(), 16 - cols)  # every row on the grid
            want = zc.layer_norm(wide, stats=True)
            assert all(torch.equal(a, b) for a, b in zip(zc.layer_norm(x, stats=True), want))
            dwant = zc.layer_norm_grad(dwide, wide, *want[1:])
            got = zc.layer_norm_grad(dy, x, *want[1:])
            assert all(torch.equal(a, b) for a, b in zip(got, dwant))
            check_norm(zc, x, None, None)


# ------------------------------------------------------------- the linear layer over its own input
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("m", [1, 2, 3, 200])
def test_int8_linear_over_its_input(zc, m, t):
    """y over x, whole or in part: x has been read by every block before any stores y (a launch of its own for it)."""
    g = gen(32)
    for k, shift in ((512, 0), (4096, 0), (1000, 7), (4096, 40)):
        layer = zc.Int8Linear.from_float(normal(g, k, k), normal(g, k))
        x = strided(normal(g, m, k).to(TYPES[t]), 64)
        start = zc.launch_count()
        want = layer(x)
        apart = zc.launch_count()
        over = layer(x, out=x._base[:, shift:shift + k])
        assert torch.equal(over, want)
        if m <= 2:
            assert apart - start == 1 and zc.launch_count() - apart == 2


def test_int8_layer_keeps_the_tensors_it_has_checked(zc):
    """Sizes, types and the pitch are looked at when a layer is made, so none of its tensors can be put in another's place."""
    g = gen(33)
    layer = zc.Int8Linear.from_float(normal(g, 40, 24), normal(g, 40))
    x = normal(g, 3, 24)
    want = layer(x)
    for name in ("weight", "scale", "bias"):
        with pytest.raises(AttributeError):
            setattr(layer, name, getattr(layer, name).half())
    assert torch.equal(layer(x), want)
    layer.bias.zero_()
    assert torch.equal(layer(x), zc.Int8Linear(layer.weight, layer.scale)(x))


def test_int8_layer_without_scales_is_refused(zc):
    with pytest.raises(zc.ZpuCudaError) as e:
        zc.Int8Linear(torch.zeros(4, 16, dtype=torch.int8, device="cuda"), None)
    assert e.value.name == "InvalidArgument"


def alone(code):
    """The output of a program of its own: a wait that runs out there is not reported here."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", "import torch, zpu_b200 as zc\nL = zc.lib()\nzc.check(L.zpucuda_init(0))\n" + code],
                       cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout.split("\n")


GIVE_UP = {"8-bit product": """
a, b, y = torch.ones(64, 64, dtype=torch.int8, device="cuda"), torch.ones(200, 64, dtype=torch.int8, device="cuda"), torch.empty(64, 200, device="cuda")
s = torch.ones(200, device="cuda")
zc.check(L.zpucuda_debug_int8_matmul(a.data_ptr(), 64, s.data_ptr(), b.data_ptr(), 64, s.data_ptr(), None, zc.F32, y.data_ptr(), 200, 64, 200, 64, 0,
                                     None, zc.stream_of()))
""", "distillation": """
x, t, i, l = torch.ones(3, 9000, device="cuda"), torch.ones(3, 2, device="cuda"), torch.ones(3, 2, dtype=torch.int64, device="cuda"), torch.empty(3, device="cuda")
zc.check(L.zpucuda_debug_distill_loss(zc.F32, x.data_ptr(), 9000, zc.F32, t.data_ptr(), 2, 3, i.data_ptr(), 2, None, 1.0, l.data_ptr(), None, 3, 9000, 2, 0,
                                      None, zc.stream_of()))
"""}


@pytest.mark.parametrize("what", list(GIVE_UP))
def test_a_wait_that_runs_out_is_reported(zc, what):
    """By zpucuda_check_device, with the kind of kernel that it ran out in."""
    before, after, text, *_ = alone("print(L.zpucuda_check_device())" + GIVE_UP[what] + "torch.cuda.synchronize()\nprint(L.zpucuda_check_device())\n"
                                    "print(L.zpucuda_last_error().decode())")
    assert before == "0" and after != "0" and what in text, (before, after, text)


def test_check_device_costs_no_more_without_the_head(zc):
    """A program that launches none of the head's kernels reads one error word as ever, not three: about a third of the
    time, and less than two thirds for sure."""
    few, many, *_ = alone("""
import time
def cost():
    t = []
    for _ in range(300):
        a = time.perf_counter()
        zc.check(L.zpucuda_check_device())
        t.append(time.perf_counter() - a)
    return sorted(t)[150]
cost()
few = cost()
x, i = torch.ones(3, 9000, device="cuda"), torch.ones(3, 2, dtype=torch.int64, device="cuda")
zc.distill_loss(x, x[:, :2].contiguous(), i)
zc.Int8Linear.from_float(x)(x)
torch.cuda.synchronize()
cost()
print(few * 1e6)
print(cost() * 1e6)
""")
    assert float(few) < 0.67 * float(many), (few, many)


def test_distill_more_rows_than_one_axis_of_a_grid(zc):
    rows = 70001
    g = gen(34)
    student, index = normal(g, rows, 5), torch.randint(0, 5, (rows, 1), generator=g, device="cuda")
    loss, d = zc.distill_value_and_grad(student, torch.zeros(rows, 1, device="cuda"), index)
    logq = torch.log_softmax(student.double(), 1)
    within(loss, -logq.gather(1, index)[:, 0], torch.full((rows,), 16 * E, device="cuda") * (1 + student.double().abs().amax(1)), "loss")
    want = logq.exp().scatter_add(1, index, torch.full((rows, 1), -1.0, dtype=torch.float64, device="cuda"))
    within(d, want, 16 * E * (1 + student.double().abs().amax(1, keepdim=True)), "dlogits")


# ------------------------------------------------------------- logits far from zero
@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("vocab", [33, 5000, 70001])
def test_distill_of_rows_at_the_lowest_value(zc, vocab, t):
    """A row of nothing but masks has equal logits: the student's distribution is even, whatever the mask's value."""
    g = gen(35)
    _, teacher, index = teach(g, 4, vocab, 7, t, ragged=False)
    student = torch.full((4, vocab), torch.finfo(TYPES[t]).min, device="cuda", dtype=TYPES[t])
    student[3] = torch.finfo(TYPES[t]).max
    for T in (0.5, 1.0, 3.0):
        lp = torch.log_softmax(teacher.double() / T, 1)
        want = T * T * (lp.exp() * (lp + math.log(vocab))).sum(1)
        d = T * torch.full((4, vocab), 1 / vocab, device="cuda", dtype=torch.float64).scatter_add(1, index, -lp.exp())
        # as for any row: roundings of log V, of each log p and of the teacher's logits, T^2 times
        size = math.log(vocab) + (lp.exp() * lp.abs()).sum(1) + (teacher.double() / T).abs().amax(1) + 4
        tol = T * T * 12 * E * size + E * want.abs()
        loss, got = zc.distill_value_and_grad(student, teacher, index, temperature=T)
        within(loss, want, tol, "loss")
        within(zc.distill_loss(student, teacher, index, temperature=T)[0], want, tol, "loss alone")
        td = T * 12 * E * size[:, None] * (1 / vocab + torch.zeros_like(d).scatter_add(1, index, lp.exp()))
        within(got, d, td + U[student.dtype] * (d.abs() + td) + S[student.dtype], "grad")


def test_distill_far_from_zero(zc):
    """Logits a long way from zero, exact there: the loss is that of the same logits about zero."""
    g = gen(36)
    student, teacher, index = teach(g, 6, 40007, 9, "f32")
    student = (student * 64).round() / 64
    want, _ = zc.distill_loss(student, teacher, index, temperature=2.0)
    for far in (-65536.0, 1024.0, 65536.0):
        loss, d = zc.distill_value_and_grad(student + far, teacher, index, temperature=2.0)
        # sums in the same order of the same differences: what is left is the listed entries' reference, a few roundings
        within(loss, want.double(), 64 * E * (1 + want.double().abs()), "loss")
        within(zc.distill_loss(student + far, teacher, index, temperature=2.0)[0], want.double(), 64 * E * (1 + want.double().abs()), "loss alone")
