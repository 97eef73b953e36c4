"""The transformer ops where their numbers or sizes lie far out: logits around
a large offset or at a mask's value, the longest rows, the most rows."""
import math

import pytest
import torch

import tensorflow_musa_extension_amd as tfma
from test_gpu_transformer import DT, U, check, gen

pytestmark = pytest.mark.gpu
ops = tfma.raw_ops


# ---------------------------------------------------------------------------
# Distillation.  With the row's maxima subtracted first,
#   loss = w T sum_j p_j ((t_j - max t) - (x_j - max x) - T (ln S_t - ln S_x)),
# so nothing is as large as the logits themselves, and the bounds below count
# roundings (units of U) of the differences alone.
# ---------------------------------------------------------------------------
def distill_bounds(logits, ids, teacher, w, t):
    """(loss, gradient, their bounds) in float64; finite logits, and at least
    one entry in every row."""
    v, k = logits.shape[-1], ids.shape[-1]
    s, w = logits.double(), w.double()
    s = s - s.amax(-1, keepdim=True)
    d = s / t
    q = d.exp()
    total = q.sum(-1, keepdim=True)
    q = q / total
    there = (ids >= 0) & (ids < v)
    at = torch.where(there, ids.long(), 0)
    r = torch.where(there, teacher.double(), -math.inf)
    r = r - r.amax(-1, keepdim=True)
    p = (r / t).exp()
    mass = p.sum(-1, keepdim=True)
    p = p / mass
    ln_x, ln_t = total.log(), mass.log()
    r = torch.where(there, r, 0.0)
    x = torch.gather(s, -1, at)
    gap = t * (ln_t - ln_x)
    term = r - x - gap
    loss = w * t * (p * term).sum(-1)
    back = q.scatter_add(-1, at, -p) * (t * w)[:, None]
    # Elements that one thread adds after the other, and the tree above it.
    n = (v / 64 if v <= 2048 else 225 + v / 1024) + 24
    # A weight is e^a with an argument of at most four roundings, six more
    # for the exponential; relative, of the sums and of p.
    e_x = (q * (4 * torch.where(q > 0, d.abs(), 0.0) + 6)).sum(-1, keepdim=True) + n
    one = 4 * r.abs() / t + 6
    e_t = (p * one).sum(-1, keepdim=True) + k / 64 + 16
    e_p = one + e_t + 2
    e_gap = t * (e_x + e_t + 4 * (ln_x.abs() + ln_t.abs())) + 4 * gap.abs()
    e_term = 3 * (r.abs() + x.abs()) + e_gap + term.abs() * (e_p + k / 64 + 18)
    el = w * t * (p * e_term).sum(-1) * U + 4 * U * loss.abs()
    e_q = q * (4 * torch.where(q > 0, d.abs(), 0.0) + 16 + e_x)
    # Weights below the smallest normal number may be 0.
    eb = (t * w)[:, None] * (e_q.scatter_add(-1, at, p * (e_p + k + 4)) * U + 1.2e-38)
    return loss.float().double(), back, el, eb


@pytest.mark.parametrize("t", [1.0, 3.0, 0.7])
@pytest.mark.parametrize("offset", [0.0, 100.0, 1e3, -1e4, 3e4])
def test_distill_of_a_student_near_its_teacher(dev, offset, t):
    """A small divergence keeps its digits wherever the logits lie."""
    rows, v = 40, 1000
    rn = gen(dev, 101)
    g = torch.Generator(device=dev).manual_seed(102)
    logits = rn(rows, v, scale=2.0) + offset
    ids = torch.stack([torch.randperm(v, generator=g, device=dev) for _ in range(rows)])
    near = torch.gather(logits, -1, ids).double() + 0.07 * rn(rows, v).double()
    w = 0.5 + rn(rows).abs()
    for teacher in (near.float(), (near - offset).float()):
        loss, back, el, eb = distill_bounds(logits, ids, teacher, w, t)
        assert bool((el < 0.05 * loss).all())  # the bound sees the loss's digits
        got = ops.MusaTopKDistillation(logits, ids, teacher, row_weights=w, temperature=t)
        check(got.loss, loss, el, "loss", torch.float32)
        check(got.backprop, back, eb, "backprop", torch.float32)


@pytest.mark.parametrize("t", [1.0, 3.0])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,v,k", [(5, 100, 9), (3, 3000, 70), (4, 8003, 20), (3, 20001, 9),
                                      (2, 50304, 64), (2, 70000, 33)])
def test_distill_around_an_offset(dev, rows, v, k, dtype, t):
    """Every width's kernel with logits around 1000."""
    rn = gen(dev, 103)
    g = torch.Generator(device=dev).manual_seed(104)
    logits = (rn(rows, v, scale=30.0) + 1000).to(DT[dtype])
    ids = torch.randint(0, v, (rows, k), generator=g, device=dev)
    teacher, w = rn(rows, k, scale=3.0, dtype=DT[dtype]), 0.5 + rn(rows).abs()
    loss, back, el, eb = distill_bounds(logits, ids, teacher, w, t)
    got = ops.MusaTopKDistillation(logits, ids, teacher, row_weights=w, temperature=t)
    check(got.loss, loss, el, "loss", torch.float32)
    check(got.backprop, back, eb, "backprop", DT[dtype])


# Masks that programs use, and the type's own lowest and largest.
MASKS = {"f32": [-1e4, -1e9, -1e30, "min", 1e30, "max"],
         "bf16": [-1e4, -1e9, -1e30, "min", 1e30, "max"], "f16": [-1e4, "min", "max"]}


@pytest.mark.parametrize("t", [1.0, 2.0, 3.0, 0.5])
@pytest.mark.parametrize("v", [100, 8003, 50304, 70000])
@pytest.mark.parametrize("dtype,value", [(d, m) for d in MASKS for m in MASKS[d]])
def test_distill_of_finite_masks(dev, dtype, value, v, t):
    """Rows that hold one finite value everywhere are uniform, whatever the
    value; rows that hold it in half of their places keep the other half's
    digits (and, where an entry lies on a mask, a loss as large as the mask)."""
    dt, rows, k = DT[dtype], 6, 12
    value = getattr(torch.finfo(dt), value) if isinstance(value, str) else value
    rn = gen(dev, 105)
    g = torch.Generator(device=dev).manual_seed(106)
    logits = rn(rows, v, scale=3.0, dtype=dt)
    ids = torch.randint(0, v, (rows, k), generator=g, device=dev)
    logits[:3] = value
    logits[3:, : v // 2] = value
    ids[3] = v - 1 - torch.arange(k, device=dev)  # none on the mask
    teacher, w = rn(rows, k, scale=3.0), 0.5 + rn(rows).abs()
    loss, back, el, eb = distill_bounds(logits, ids, teacher, w, t)
    got = ops.MusaTopKDistillation(logits, ids, teacher, row_weights=w, temperature=t)
    check(got.loss, loss, el, "loss", torch.float32)
    check(got.backprop, back, eb, "backprop", dt)


@pytest.mark.parametrize("t", [0.5, 0.25, 2.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distill_of_a_finitely_masked_teacher(dev, dtype, t):
    """An entry at the type's lowest value is there: it has no weight beside
    larger ones, and a row of such entries is uniform."""
    dt, rows, v, k = DT[dtype], 4, 300, 8
    rn = gen(dev, 107)
    logits, teacher, w = rn(rows, v, dtype=dt), rn(rows, k, dtype=dt), 0.5 + rn(rows).abs()
    ids = torch.arange(rows * k, device=dev).reshape(rows, k)
    low = torch.finfo(dt).min
    teacher[0] = low
    teacher[1, 3:] = low
    teacher[2] = -low
    teacher[3, 0] = -low
    loss, back, el, eb = distill_bounds(logits, ids, teacher, w, t)
    got = ops.MusaTopKDistillation(logits, ids, teacher, row_weights=w, temperature=t)
    check(got.loss, loss, el, "loss", torch.float32)
    check(got.backprop, back, eb, "backprop", dt)


@pytest.mark.parametrize("t", [1e-3, 1e-30, 1e-39, 1e-45])
def test_distill_at_the_smallest_temperatures(dev, t):
    """The softmax is its maximum's place; no 0 meets an infinity."""
    v = 500
    logits = gen(dev, 108)(2, v)
    logits[:, 7] = 20
    ids = torch.tensor([[7, 3], [7, 9]], device=dev)
    teacher = torch.tensor([[3.0, -8.0], [-8.0, 3.0]], device=dev)
    got = ops.MusaTopKDistillation(logits, ids, teacher, temperature=t)
    # The teacher's place is the student's in one row and 20 - x[9] below its
    # largest in the other: loss T (20 - x[9]).
    want = float(torch.tensor(t)) * (20 - float(logits[1, 9]))
    assert float(got.loss[0]) == 0 and abs(float(got.loss[1]) - want) <= 4 * U * want + 2.0 ** -149
    back = torch.zeros(2, v, device=dev)
    back[1, 7], back[1, 9] = float(torch.tensor(t)), -float(torch.tensor(t))
    assert torch.equal(got.backprop, back)


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------
def sparse_places(dev, k, n, seed):
    """n places of [0, k): the first, the last, those around every quarter and
    others as they fall."""
    g = torch.Generator(device=dev).manual_seed(seed)
    fixed = [q * k // 4 + d for q in range(1, 4) for d in (-1, 0)] + [0, 1, k - 2, k - 1]
    rest = torch.randint(0, k, (n - len(fixed),), generator=g, device=dev)
    return torch.cat([torch.tensor(fixed, device=dev), rest]).unique()


@pytest.mark.parametrize("tile", [0, 1, 2, 3, None])
def test_linear_quantized_longest_rows(dev, tune, tile):
    """Rows of 8 MiB, 256 of a tile: their offsets pass 2^31 by nothing.  x is
    zero but for some hundred whole numbers a row, w is -1, 0 and 1: sums that
    every order of them holds exactly."""
    m, k, n = 256, 1 << 23, 256
    if tile is not None:
        tune("linear_tile", tile)
        tune("linear_splits", 8)
    g = torch.Generator(device=dev).manual_seed(110)
    at = sparse_places(dev, k, 200, 111)
    some = torch.randint(-2, 3, (m, at.numel()), generator=g, device=dev).float()
    x = torch.zeros(m, k, dtype=torch.uint8, device=dev)
    x[:, at] = some.to(torch.float8_e4m3fn).view(torch.uint8)
    w = torch.randint(0, 3, (n, k), generator=g, device=dev, dtype=torch.uint8)
    w = torch.where(w == 2, 0xB8, w * 0x38).to(torch.uint8).view(torch.float8_e4m3fn)
    one = torch.ones(n, device=dev)
    got = ops.MusaLinearQuantized(x.view(torch.float8_e4m3fn), one, w, one, out_type=torch.float16)
    want = some.double() @ w.view(torch.uint8)[:, at].view(torch.float8_e4m3fn).double().T
    assert float(want.std()) > 5
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("tb", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_of_rows_over_4_mib(dev, dtype, tb):
    """The kernel of the longest rows, with operands of more than 2^31 bytes,
    at whole numbers whose sums are exact."""
    dt = DT[dtype]
    long = (1 << 22) // dt.itemsize + 72
    g = torch.Generator(device=dev).manual_seed(112)
    if tb:  # both operands' rows, and a long sum
        m, k, n = 520, long, 520
        at = sparse_places(dev, k, 100, 113)
        some = torch.randint(-2, 3, (m, at.numel()), generator=g, device=dev).to(dt)
        x = torch.zeros(m, k, dtype=dt, device=dev)
        x[:, at] = some
        w = torch.randint(-1, 2, (n, k), generator=g, device=dev, dtype=torch.int8).to(dt)
        want = some.double() @ w[:, at].double().T
    else:  # w's rows
        m, k, n = 40, 520, long
        x = torch.randint(-2, 3, (m, k), generator=g, device=dev).to(dt)
        x[:, torch.rand(k, generator=g, device=dev) < 0.8] = 0
        w = torch.randint(-1, 2, (k, n), generator=g, device=dev, dtype=torch.int8).to(dt)
        want = (x.float() @ w.float()).double()  # whole numbers below 2^24
    assert float(want.std()) > 5 and float(want.abs().max()) <= 256
    got = ops.MusaLinear(x, w, transpose_b=tb).y
    assert ops.last_kernel_name() == "tfma_linear"
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("shape,few", [
    ((1, 16, 1), True), ((1, 512, 4096), True), ((4, 1536, 300), True), ((3, 1040, 70), True),
    ((16, 512, 4096), True), ((13, 400, 75), True), ((5, 16, 4095), True),
    ((1, 512, 4097), False), ((4, 1552, 300), False), ((5, 528, 70), False), ((16, 1024, 1024), False),
    ((1, 2048, 8192), False), ((16, 2048, 2048), False), ((16, 4096, 4096), False),
    ((16, 4096, 8192), False), ((9, 4096, 72), False)])
def test_linear_quantized_of_few_tokens(dev, shape, few):
    """Either kernel on its side of the rule, at whole numbers whose sums are
    exact."""
    m, k, n = shape
    g = torch.Generator(device=dev).manual_seed(114)
    x = torch.randint(-2, 3, (m, k), generator=g, device=dev)
    x[torch.rand(m, k, generator=g, device=dev) < max(0.0, 1 - 200 / k)] = 0
    w = torch.randint(-1, 2, (n, k), generator=g, device=dev)
    xs = 2.0 ** torch.randint(-2, 3, (m,), generator=g, device=dev)
    ws = 2.0 ** torch.randint(-2, 3, (n,), generator=g, device=dev)
    f8 = torch.float8_e4m3fn
    got = ops.MusaLinearQuantized(x.to(f8), xs, w.to(f8), ws, out_type=torch.float16)
    assert (ops.last_kernel_name() == "tfma_linear_few") == few
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    assert torch.equal(got.double(), want)


# ---------------------------------------------------------------------------
# More threads than a grid's dimension counts: rows of few elements (and the
# longest rows) in numbers that take more than 2^32.
# ---------------------------------------------------------------------------
def some_rows(dev, rows, of_a_grid):
    """Rows at both ends, on both sides of `of_a_grid` and in between."""
    g = torch.Generator(device=dev).manual_seed(120)
    some = torch.randint(0, rows, (40,), generator=g, device=dev)
    ends = [0, 1, 19, 20, of_a_grid - 1, of_a_grid, rows - 2, rows - 1]
    return torch.cat([torch.tensor(ends, device=dev), some])


def test_norm_of_more_rows_than_a_grid_counts(dev):
    rows, c = (1 << 26) + 77, 8
    x = torch.empty(rows, c, dtype=torch.bfloat16, device=dev)
    x.normal_(generator=torch.Generator(device=dev).manual_seed(121))
    gamma = torch.ones(c, device=dev)
    out = ops.MusaAddRmsNormResult(torch.full_like(x, math.nan), x,
                                   torch.full((rows,), math.nan, device=dev))
    ops.MusaAddRmsNorm(x, gamma, out=out)
    assert not bool(out.rstd.isnan().any()) and not bool(out.y.isnan().any())
    pick = some_rows(dev, rows, 1 << 26)
    want = ops.MusaAddRmsNorm(x[pick], gamma)
    assert torch.equal(out.y[pick], want.y) and torch.equal(out.rstd[pick], want.rstd)
    q = ops.MusaAddRmsNormQuantizedResult(torch.zeros(rows, c, dtype=torch.float8_e4m3fn, device=dev),
                                          out.rstd.fill_(math.nan), x)
    ops.MusaAddRmsNormQuantized(x, gamma, out=q)
    assert not bool(q.scale.isnan().any())
    wq = ops.MusaAddRmsNormQuantized(x[pick], gamma)
    assert torch.equal(q.y.view(torch.uint8)[pick], wq.y.view(torch.uint8))


def test_norm_of_more_wide_rows_than_a_grid_counts(dev):
    """A workgroup a row, over the input's own memory."""
    rows, c = (1 << 24) + 77, 1032
    x = torch.empty(rows, c, dtype=torch.bfloat16, device=dev)
    x.normal_(generator=torch.Generator(device=dev).manual_seed(122))
    gamma = torch.ones(c, device=dev)
    pick = some_rows(dev, rows, 1 << 24)
    want = ops.MusaAddRmsNorm(x[pick], gamma)
    rstd = torch.full((rows,), math.nan, device=dev)
    ops.MusaAddRmsNorm(x, gamma, out=ops.MusaAddRmsNormResult(x, x, rstd))
    assert not bool(rstd.isnan().any())
    assert torch.equal(x[pick], want.y) and torch.equal(rstd[pick], want.rstd)


def test_norm_grad_of_the_longest_rows(dev):
    """gamma's gradient has more columns than a grid counts."""
    rows, c = 6, (1 << 28) + 136
    g = torch.Generator(device=dev).manual_seed(123)
    h = torch.empty(rows, c, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    gamma = torch.ones(c, device=dev)
    rstd = torch.ones(rows, device=dev)
    out = ops.MusaAddRmsNormGradResult(torch.empty_like(h), torch.full((c,), math.nan, device=dev))
    ops.MusaAddRmsNormGrad(h, h, gamma, rstd, out=out)
    assert not bool(out.gamma_backprop.isnan().any())
    last = slice(c - 200, c)
    for at in (slice(0, 200), slice(c // 2, c // 2 + 200), last):
        want = h[:, at].double().square()
        check(out.gamma_backprop[at], want.sum(0), want.sum(0) * (rows + 4) * U, "dgamma")


def test_distill_of_more_rows_than_a_grid_counts(dev):
    rows, v, k = (1 << 26) + 77, 9, 2
    g = torch.Generator(device=dev).manual_seed(124)
    logits = torch.empty(rows, v, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    ids = torch.randint(0, v, (rows, k), generator=g, device=dev, dtype=torch.int32)
    teacher = torch.empty(rows, k, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    out = ops.MusaTopKDistillationResult(torch.full((rows,), math.nan, device=dev),
                                         torch.full_like(logits, math.nan))
    ops.MusaTopKDistillation(logits, ids, teacher, out=out)
    assert not bool(out.loss.isnan().any()) and not bool(out.backprop.isnan().any())
    pick = some_rows(dev, rows, 1 << 26)
    want = ops.MusaTopKDistillation(logits[pick], ids[pick], teacher[pick])
    assert torch.equal(out.loss[pick], want.loss) and torch.equal(out.backprop[pick], want.backprop)


def test_linear_copies_of_more_rows_than_a_grid_counts(dev):
    """Ragged rows, copied to whole vectors first."""
    m, k, n = (1 << 26) + 77, 9, 8
    g = torch.Generator(device=dev).manual_seed(125)
    x = torch.randint(-2, 3, (m, k), generator=g, device=dev, dtype=torch.int8).bfloat16()
    w = torch.randint(-1, 2, (k, n), generator=g, device=dev).bfloat16()
    y = ops.MusaLinear(x, w).y
    assert torch.equal(y, (x.float() @ w.float()).bfloat16())  # whole numbers


@pytest.mark.parametrize("tb", [False, True])
def test_linear_of_one_row_and_the_most_columns(dev, tb):
    """A product of few rows whose columns take more threads than a grid
    counts, with either order of w."""
    k, n = (3, (1 << 27) + 72) if tb else (1, (1 << 28) + 72)
    g = torch.Generator(device=dev).manual_seed(126)
    w = torch.randint(-1, 2, (n, k) if tb else (k, n), generator=g, device=dev, dtype=torch.int8).half()
    x = torch.tensor([[2.0, -1.0, 3.0][:k]], device=dev).half()
    out = ops.MusaLinearResult(torch.full((1, n), math.nan, dtype=torch.float16, device=dev), None)
    ops.MusaLinear(x, w, transpose_b=tb, out=out)
    assert ops.last_kernel_name() == "tfma_linear_few"
    want = (w.float() * x[0].float()).sum(1) if tb else w[0].float() * 2
    assert torch.equal(out.y[0], want.half())
