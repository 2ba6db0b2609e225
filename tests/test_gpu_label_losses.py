"""GPU tests of the label losses (kge/label_losses.py, csrc/label_loss.hip) against their formulas in
64 bits on the CPU.

Tolerances (u = 2^-24, half a step of fp32).  The kernel's exponentials are exp2((s - M) k2) with three
roundings in the argument (difference, product, k2) and one step (2 u) in the result, so relative to its
own size a term is off by at most e_j = 3 u |s_j - M| / tau + 2 u; a thread adds at most K = m / 64 + 16
terms one after the other before fp64 takes over (64 threads at least share a row), each addition
rounding by u.  Hence
    |d log Z| <= E = sum_j p_j e_j + (K + 4) u,       |d l| <= E + u |l|   (the result's own rounding).
A gradient entry c / tau ([j = y] - p_j): |d| <= |c| / tau (p_j (e_j + E + 4 u)) + |dc| / tau + 2 u |value|
and half a step of a 16-bit output type.  dc follows from dl through the coefficient's slope."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
SUB = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}  # flushed / subnormal step


@pytest.fixture(scope="module")
def engine():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from kge import _lib, engine
    _lib.lib()
    return engine


def block(n, m, dtype, seed, ld=None, offset=0, masked=True, std=2.0):
    """Scores [n, m] of row stride ld (m if None) starting `offset` elements into their storage,
    with masked columns, label -1 rows and the labels of the others anywhere (column 0 and m - 1 too)."""
    g = torch.Generator().manual_seed(seed)
    ld = ld or m
    flat = torch.full((offset + n * ld + 16,), 77.0, dtype=dtype)
    s = flat[offset:offset + n * ld].view(n, ld)[:, :m]
    s.copy_((torch.randn(n, m, generator=g) * std).to(dtype))
    y = torch.randint(0, m, (n,), generator=g)
    y[0] = m - 1
    if n > 1:
        y[1] = 0
    if masked and m > 4:
        hide = torch.rand(n, m, generator=g) < 0.05
        hide.scatter_(1, y[:, None], False)
        s.masked_fill_(hide, -math.inf)
    if n > 2:
        y[2::7] = -1
    dev = flat.cuda()
    return dev[offset:offset + n * ld].view(n, ld)[:, :m], y.cuda()


def formulas(s, y, tau):
    """(l, p, e, E) in 64 bits on the CPU: log-probabilities, probabilities and the bounds above."""
    x = s.detach().cpu().double() / tau
    y = y.cpu()
    mx = x.amax(1, keepdim=True)
    p = torch.softmax(x, 1)
    gap = torch.where(p > 0, (x - mx).abs(), 0.0)
    e = 3 * U * gap + 2 * U
    E = (p * e).sum(1) + (s.shape[1] / 64 + 20) * U
    # (x - max) - log sum: a row of the type's lowest value would absorb log m in max + log sum
    l = (x - mx).gather(1, y.clamp(min=0)[:, None])[:, 0] - torch.exp(x - mx).sum(1).log()
    l = torch.where(y >= 0, l, 0.0)
    return l, p, e, E


def check_logp(got, l, E, y):
    err = (got.detach().cpu().double() - l).abs()
    tol = torch.where(y.cpu() >= 0, E + U * l.abs(), 0.0)
    assert (err <= tol).all(), (err - tol).max()


def check_grad(got, s, y, tau, c, dc, p, e, E):
    onehot = torch.zeros_like(p)
    yc = y.cpu()
    onehot[torch.arange(len(yc))[yc >= 0], yc[yc >= 0]] = 1.0
    c = torch.where(yc >= 0, c, 0.0)
    want = c[:, None] / tau * (onehot - p)
    want[yc < 0] = 0.0
    bound = c.abs()[:, None] / tau * p * (e + E[:, None] + 4 * U) + dc[:, None] / tau * (onehot - p).abs() + 2 * U * want.abs()
    tol = bound + (HALF[s.dtype] * (want.abs() + bound) + SUB[s.dtype])
    assert got.dtype == s.dtype and got.shape == s.shape
    err = (got.detach().cpu().double() - want).abs()
    assert torch.isfinite(got.float()).all()
    assert (err <= tol).all(), ((err - tol).max(), err.max())
    assert (got.cpu()[yc < 0] == 0).all()
    return want


SHAPES = [  # n, m, row stride, storage offset
    (1, 1, None, 0), (1, 2, None, 1), (3, 7, None, 0), (5, 8, 8, 0), (9, 130, None, 3), (17, 1001, 1009, 5),
    (64, 500, 504, 0), (4, 14541, None, 0), (300, 4099, 4104, 0), (2, 70001, None, 1), (3, 300000, 300008, 0),
    (2100, 33, None, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n, m, ld, offset", SHAPES)
def test_label_logprobs_and_gradient(engine, n, m, ld, offset, dtype):
    tau = 0.7 if n % 2 else 1.0
    s, y = block(n, m, dtype, n * 31 + m, ld, offset)
    s.requires_grad_(True)
    logp = engine.label_logprobs(s, y, tau)
    l, p, e, E = formulas(s, y, tau)
    check_logp(logp, l, E, y)
    g = torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    (grad,) = torch.autograd.grad(logp, s, g)
    check_grad(grad, s, y, tau, g.cpu().double(), torch.zeros(n, dtype=torch.float64), p, e, E)
    with torch.no_grad():  # the form without a gradient: the same numbers
        assert torch.equal(engine.label_logprobs(s, y, tau), logp)


def policy_inputs(l, y, seed):
    """Old and reference log-probabilities around l; no ratio within 1e-3 of a border of [0.8, 1.28]."""
    g = torch.Generator().manual_seed(seed)
    n = l.numel()
    step = torch.randn(n, generator=g).double() * 0.3
    for b in (math.log(0.8), math.log(1.28)):
        step = torch.where((step - b).abs() < 1e-3, step + 4e-3, step)
    old = (l - step).float()
    ref = (l + torch.randn(n, generator=g).double() * 0.3).float()
    adv = torch.randn(n, generator=g)
    adv[n // 2] = 0.0
    w = torch.rand(n, generator=g) + 0.5
    return old, ref, adv, w


def policy_formula(l, y, old, ref, adv, w, kl, scale):
    """(loss, c, |dc/dl|, |dloss/dl|) in 64 bits."""
    old, adv, w = old.double(), adv.double(), w.double()
    r = torch.exp(l - old)
    held = r.clamp(0.8, 1.28) * adv
    rows, c, slope = -torch.minimum(r * adv, held), torch.where(r * adv <= held, -r * adv, 0.0), (r * adv).abs()
    if ref is not None:
        d = ref.double() - l
        rows, c, slope = rows + kl * (torch.expm1(d) - d), c - kl * torch.expm1(d), slope + kl * torch.exp(d)
    w = torch.where(y.cpu() >= 0, w * scale, 0.0)
    return (w * rows).sum(), w * c, w * slope, w * (r * adv).abs() + w * (kl * 2 if ref is not None else 0.0), (w * rows).abs()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n, m, ld, offset", SHAPES)
@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_policy_loss(engine, n, m, ld, offset, dtype, kl):
    tau = 1.3 if n % 2 else 1.0
    s, y = block(n, m, dtype, n * 17 + m, ld, offset)
    l, p, e, E = formulas(s, y, tau)
    old, ref, adv, w = policy_inputs(l, y, n + m)
    scale = 8.0 / n
    want, c, slope, steep, rows = policy_formula(l, y, old, ref if kl else None, adv, w, kl, scale)
    dl = E + U * 0  # the kernel keeps l in 64 bits between the rows and the coefficients
    dc = slope * dl * 1.01 + 2 * U * c.abs()
    dloss = float((steep * dl * 1.01).sum() + 2 * U * abs(float(want)) + 1e-12)
    args = (adv.cuda(), old.cuda(), ref.cuda())
    kw = dict(clip=(0.2, 0.28), kl=kl, temperature=tau, weights=w.cuda(), scale=scale)
    loss, logp, grad = engine.policy_loss_grad(s, y, *args, **kw)
    check_logp(logp, l, E, y)
    assert abs(float(loss) - float(want)) <= dloss
    check_grad(grad, s, y, tau, c, dc, p, e, E)
    # under autograd, with an upstream factor
    leaf = s.detach().requires_grad_(True)
    loss2, logp2 = engine.policy_loss(leaf, y, *args, **kw)
    check_logp(logp2, l, E, y)  # (the two forms group their sums differently: the same bound, not the same bits)
    assert not logp2.requires_grad
    assert abs(float(loss2.detach()) - float(want)) <= dloss
    (g2,) = torch.autograd.grad(loss2 * 0.5, leaf)
    check_grad(g2, s, y, tau, 0.5 * c, 0.5 * dc + U * c.abs(), p, e, E)
    # in place of the scores
    own = s.clone() if ld is None else None
    if own is not None:
        loss3, _, g3 = engine.policy_loss_grad(own, y, *args, out=own, **kw)
        # (a clone may be aligned otherwise, which groups the sums otherwise: the same bound, not the same bits)
        assert g3.data_ptr() == own.data_ptr() and abs(float(loss3) - float(want)) <= dloss
        check_grad(g3, s, y, tau, c, dc, p, e, E)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("lens, m, ld, offset", [
    ([1, 1], 5, None, 0), ([1, 1] * 8, 14541, 14544, 0), ([3, 0, 0, 0, 1, 70, 2, 5], 333, None, 1),
    ([2, 4, 1, 9, 12, 3], 30011, None, 0), ([130, 1, 1, 130], 64, 72, 8)])
def test_preference_loss(engine, lens, m, ld, offset, average, dtype):
    n = sum(lens) + 3  # one row before the first sequence, two behind the last
    pairs, beta, eps, scale, tau = len(lens) // 2, 0.3, 0.1, 4.0 / (len(lens) // 2), 0.9
    s, y = block(n, m, dtype, n + m, ld, offset)
    y[1] = 0
    l, p, e, E = formulas(s, y, tau)
    ptr = torch.tensor([1] + lens).cumsum(0)
    has = (y.cpu() >= 0).double()
    seq_of = torch.full((n,), -1)
    for q in range(2 * pairs):
        seq_of[ptr[q]:ptr[q + 1]] = q
    inside = seq_of >= 0
    count = torch.zeros(2 * pairs, dtype=torch.float64).index_add_(0, seq_of[inside], has[inside])
    div = count.clamp(min=1) if average else torch.ones_like(count)
    sums = lambda v: torch.zeros(2 * pairs, dtype=torch.float64).index_add_(0, seq_of[inside], (v * has)[inside]) / div  # noqa: E731
    pi, dpi = sums(l), sums(E + U * l.abs())  # the rows' l are held in fp32
    ref = (pi + torch.randn(2 * pairs, generator=torch.Generator().manual_seed(3)).double()).float()
    h = pi - ref.double()
    z = beta * (h[0::2] - h[1::2])
    dz = beta * (dpi[0::2] + dpi[1::2])
    logsig = torch.nn.functional.logsigmoid
    want = -scale * ((1 - eps) * logsig(z) + eps * logsig(-z)).sum()
    c = -scale * beta * ((1 - eps) - torch.sigmoid(z))
    per_seq = torch.stack([c, -c], 1).view(-1) / div
    dper = torch.stack([scale * beta * dz / 4] * 2, 1).view(-1) / div
    coef, dc = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    coef[inside], dc[inside] = per_seq[seq_of[inside]], dper[seq_of[inside]]
    dc = dc * 1.01 + 2 * U * coef.abs()
    kw = dict(beta=beta, smoothing=eps, average=average, temperature=tau, scale=scale)
    loss, seq, grad = engine.preference_loss_grad(s, y, ptr.cuda(), ref.cuda(), **kw)
    dloss = float(scale * dz.sum() * 1.01 + 2 * U * abs(want))
    assert abs(float(loss) - float(want)) <= dloss
    assert ((seq.cpu().double() - pi).abs() <= dpi + U * pi.abs()).all()
    check_grad(grad, s, y, tau, coef, dc, p, e, E)
    assert (grad[0] == 0).all() and (grad[-2:] == 0).all()
    leaf = s.detach().requires_grad_(True)
    loss2, seq2 = engine.preference_loss(leaf, y, ptr.cuda(), ref.cuda(), **kw)
    assert torch.equal(seq, seq2) and torch.equal(loss, loss2)
    (2.0 * loss2).backward()
    check_grad(leaf.grad, s, y, tau, 2 * coef, 2 * dc + 2 * U * coef.abs(), p, e, E)
    # no reference: zeros
    a = engine.preference_loss(s, y, ptr.cuda(), None, **kw)[0]
    b = engine.preference_loss(s, y, ptr.cuda(), torch.zeros(2 * pairs, device="cuda"), **kw)[0]
    assert torch.equal(a, b)


def test_gradients_against_differences(engine):
    """Central differences of the losses in 64 bits (the formula's own) and of the kernel's loss."""
    n, m = 6, 23
    s, y = block(n, m, torch.float32, 5, masked=False, std=1.0)
    l, p, _, _ = formulas(s, y, 1.0)
    old, ref, adv, w = policy_inputs(l, y, 9)
    ptr = torch.tensor([0, 1, 3, 5, 6]).cuda()
    calls = [lambda t: engine.policy_loss(t, y, adv.cuda(), old.cuda(), ref.cuda(), kl=0.2, weights=w.cuda())[0],
             lambda t: engine.preference_loss(t, y, ptr, None, beta=0.5)[0],
             lambda t: (engine.label_logprobs(t, y) * w.cuda()).sum()]
    h = 2.0 ** -6
    for call in calls:
        leaf = s.detach().clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(call(leaf), leaf)
        for i, j in ((0, m - 1), (0, 3), (1, 0), (3, 7), (4, 11), (5, int(y[5]))):
            up, down = s.clone(), s.clone()
            up[i, j] += h
            down[i, j] -= h
            with torch.no_grad():
                diff = (float(call(up)) - float(call(down))) / (2 * h)
            # third derivative of these losses is below 8 here: h^2 / 6 * 8; fp32 losses up to 64: 2 u 64 / 2h
            assert abs(diff - float(grad[i, j])) <= h * h / 6 * 8 + 64 * 2 * U / (2 * h), (i, j)


def test_empty_blocks_and_rows_without_labels(engine):
    for dtype in (torch.float32, torch.bfloat16):
        s = torch.zeros(0, 9, device="cuda", dtype=dtype)
        y = torch.zeros(0, device="cuda", dtype=torch.int64)
        v = torch.zeros(0, device="cuda")
        assert engine.label_logprobs(s, y).shape == (0,)
        loss, logp, grad = engine.policy_loss_grad(s, y, v, v)
        assert float(loss) == 0 and logp.shape == (0,) and grad.shape == (0, 9)
        ptr = torch.zeros(3, device="cuda", dtype=torch.int64)
        loss, seq, grad = engine.preference_loss_grad(s, y, ptr)
        assert abs(float(loss) - math.log(2.0)) <= 2 * U and (seq == 0).all()
        # all rows unlabelled: nothing is read (NaN scores), everything is zero
        s = torch.full((5, 9), math.nan, device="cuda", dtype=dtype)
        y = torch.full((5,), -1, device="cuda")
        v = torch.ones(5, device="cuda")
        loss, logp, grad = engine.policy_loss_grad(s, y, v, v, v, kl=0.1)
        assert float(loss) == 0 and (logp == 0).all() and (grad == 0).all()
        # no pairs: no loss, zero gradient
        loss, seq, grad = engine.preference_loss_grad(s, torch.zeros_like(y), ptr[:1])
        assert float(loss) == 0 and seq.numel() == 0 and (grad == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [40, 20001])
def test_infinities_and_nan(engine, dtype, m):
    """-inf everywhere but the label: certainty.  -inf in whole parts of a row: as if they were not
    there.  The type's lowest value likewise.  NaN, +inf, or nothing but -inf: NaN in that row alone."""
    s, y = block(8, m, dtype, 3, masked=False)
    y = torch.arange(8, device="cuda") % m
    low = torch.finfo(dtype).min
    s[0] = -math.inf
    s[0, 0] = 1.5
    s[1, m // 2:] = -math.inf
    s[2, m // 2:] = low
    s[3] = -math.inf
    s[4, m - 1] = math.nan
    s[5, 9] = math.inf
    s[6] = low
    logp = engine.label_logprobs(s, y)
    l, p, e, E = formulas(s, y, 1.0)
    good = torch.tensor([0, 1, 2, 6, 7])
    assert float(logp[0]) == 0.0
    err = (logp.cpu().double() - l).abs()[good]
    assert (err <= (E + U * l.abs())[good]).all()
    assert torch.isnan(logp[3]) and torch.isnan(logp[4]) and torch.isnan(logp[5])
    v = torch.ones(8, device="cuda")
    loss, _, grad = engine.policy_loss_grad(s, y, v, l.float().nan_to_num().cuda(), scale=1.0)
    assert torch.isnan(loss)
    rows_nan = torch.isnan(grad.float()).any(1).cpu()
    assert rows_nan.tolist() == [False, False, False, True, True, True, False, False]
    assert (grad[1, m // 2:] == 0).all() and (grad[2, m // 2:] == 0).all()


def test_labels_out_of_range_poison_their_row_only(engine, monkeypatch):
    from kge import _lib as L
    monkeypatch.setattr(L, "CHECK_INDEX", False)
    s, _ = block(4, 50, torch.float32, 1, masked=False)
    y = torch.tensor([3, 50, -2, 49], device="cuda")
    assert torch.isnan(engine.label_logprobs(s, y)).tolist() == [False, True, True, False]
    v = torch.ones(4, device="cuda")
    loss, _, grad = engine.policy_loss_grad(s, y, v, v)
    assert torch.isnan(loss)
    assert torch.isnan(grad).all(1).tolist() == [False, True, True, False]
    assert torch.isnan(grad).any(1).tolist() == [False, True, True, False]
    # sequence bounds beyond the rows are cut off there
    y = torch.tensor([3, 2, 1, 49], device="cuda")
    a = engine.preference_loss(s, y, torch.tensor([-5, 1, 99], device="cuda"))[1]
    b = engine.preference_loss(s, y, torch.tensor([0, 1, 4], device="cuda"))[1]
    assert torch.equal(a, b)


def test_extreme_ratios_and_margins(engine):
    """Far-off policies and margins: no overflow where the formula has none, and its infinities where it has."""
    s, y = block(4, 64, torch.float32, 2, masked=False)
    y = torch.tensor([1, 2, 3, 4], device="cuda")
    l = formulas(s, y, 1.0)[0]
    old = (l + torch.tensor([200.0, -200.0, 0.0, 0.0])).float().cuda()
    ref = (l + torch.tensor([0.0, 0.0, -300.0, 0.0])).float().cuda()
    adv = torch.tensor([1.0, 1.0, 1.0, -1.0], device="cuda")
    loss, _, grad = engine.policy_loss_grad(s, y, adv, old, ref, kl=1.0)
    # rows: -(e^-200), -1.2 (clipped), -1 + (e^-300 + 300 - 1), +1
    assert abs(float(loss) - (-1.2 - 1.0 + 299.0 + 1.0)) <= 1e-3  # d of 300 comes from fp32 inputs: 300 u each side
    assert torch.isfinite(grad).all() and (grad[1].abs() <= 1e-5).all()
    ptr = torch.arange(5, device="cuda")
    ref = torch.tensor([3000.0, 0.0, -3000.0, 0.0], device="cuda")
    loss, _, grad = engine.preference_loss_grad(s, y, ptr, ref, beta=1.0)
    assert abs(float(loss) - 3000.0) < 20 and torch.isfinite(grad).all()
    assert float(grad[2].abs().max()) == 0.0 and float(grad[0].abs().max()) > 0.5


def test_arguments_that_need_a_copy(engine):
    """Transposed, expanded and strided inputs, int32 labels, bf16 and expanded vectors."""
    s, y = block(6, 40, torch.float32, 4, masked=False)
    want = engine.label_logprobs(s, y)
    assert torch.equal(engine.label_logprobs(s.t().contiguous().t(), y), want)
    wide = torch.zeros(6, 80, device="cuda")
    wide[:, ::2] = s
    assert torch.equal(engine.label_logprobs(wide[:, ::2], y.int()), want)
    one = engine.label_logprobs(s[:1].expand(6, 40), y[:1].expand(6))
    assert (one == want[0]).all()
    adv = torch.ones(1, device="cuda").expand(6)
    old = want.detach()
    a = engine.policy_loss(s, y, adv, old)[0]
    b = engine.policy_loss(s, y, adv.bfloat16(), old)[0]
    assert torch.equal(a, b)
    # an expanded leaf collects the gradients of all its rows
    leaf = s[:1].clone().requires_grad_(True)
    loss = engine.label_logprobs(leaf.expand(6, 40), torch.arange(6, device="cuda")).sum()
    (g,) = torch.autograd.grad(loss, leaf)
    p = torch.softmax(s[0].cpu().double(), 0)
    ref = torch.cat([torch.ones(6), torch.zeros(34)]).double() - 6 * p
    assert ((g[0].cpu().double() - ref).abs() <= 6 * 40 * U).all()


def test_out_refusals(engine):
    s, y = block(4, 40, torch.float32, 4, masked=False)
    v = torch.ones(4, device="cuda")
    flat = torch.zeros(200, device="cuda")
    s2 = flat[:160].view(4, 40)
    for scores, out in ((s, torch.zeros(4, 41, device="cuda")), (s, torch.zeros(4, 40, device="cuda").half()),
                        (s, torch.zeros(4, 40)), (s, torch.zeros(40, 4, device="cuda").t()),
                        (s2, flat[8:168].view(4, 40)), (s, s[:1].expand(4, 40))):
        with pytest.raises(ValueError, match="out"):
            engine.policy_loss_grad(scores, y, v, v, out=out)
    # the upper half of a buffer beside scores in the lower half is fine
    flat = torch.zeros(320, device="cuda")
    flat[:160] = s.reshape(-1)
    g = engine.policy_loss_grad(flat[:160].view(4, 40), y, v, v, out=flat[160:].view(4, 40))[2]
    assert torch.equal(g, engine.policy_loss_grad(s, y, v, v)[2])
    # an output of another alignment than the scores
    other = torch.zeros(4 * 40 + 3, device="cuda")[3:].view(4, 40)
    assert torch.equal(engine.policy_loss_grad(s, y, v, v, out=other)[2], g)


@pytest.mark.parametrize("n, m", [(16, 500), (3, 50001)])
def test_recorded_in_a_graph(engine, n, m):
    """Each entry point recorded once and replayed on new contents, with eager work in between; two
    recorded graphs do not share a workspace."""
    s, y = block(n, m, torch.float32, 1, masked=False)
    v = torch.ones(n, device="cuda")
    ptr = torch.tensor([0, 1, n], device="cuda")

    def work():
        leaf = s.detach().requires_grad_(True)
        logp = engine.label_logprobs(leaf, y)
        (g0,) = torch.autograd.grad(logp, leaf, v)
        return [logp.detach(), g0, *engine.policy_loss_grad(s, y, v, old, ref, kl=0.1),
                *engine.preference_loss_grad(s, y, ptr)]

    old = engine.label_logprobs(s, y) + 0.05
    ref = old - 0.1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work()
        graphs.append((graph, outs))
    for k in range(4):
        s.copy_(block(n, m, torch.float32, 50 + k, masked=False)[0])  # (a mask would hide labels of y)
        want = [t.clone() for t in work()]
        torch.cuda.synchronize()
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_two_streams_at_once(engine):
    """Calls that overlap on two streams give the same bits as one after the other."""
    data = [block(40, 20011, torch.float32, k) for k in range(2)]
    want = [engine.policy_loss_grad(s, y, torch.ones(40, device="cuda"), torch.full((40,), -9.0, device="cuda"))
            for s, y in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for rep in range(5):
        for k, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                s, y = data[k]
                got[k] = engine.policy_loss_grad(s, y, torch.ones(40, device="cuda"),
                                                 torch.full((40,), -9.0, device="cuda"))
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))


def test_rows_past_32_bit_offsets(engine):
    """A bf16 block of more than 2^32 bytes and 2^31 elements: the last rows are addressed in 64 bits."""
    n, m = 2200, 1000003
    s = torch.zeros(n, m, device="cuda", dtype=torch.bfloat16)
    rows = [0, 1, 1100, n - 1]
    g = torch.Generator(device="cuda").manual_seed(0)
    for i in rows:
        s[i] = torch.randn(m, device="cuda", generator=g).bfloat16()
    y = torch.full((n,), -1, device="cuda")
    y[rows] = torch.tensor([m - 1, 0, 77, m - 2], device="cuda")
    logp = engine.label_logprobs(s, y)
    l, p, e, E = formulas(s[rows], y[rows], 1.0)
    check_logp(logp[rows], l, E, y[rows])
    v = torch.ones(n, device="cuda")
    loss, _, grad = engine.policy_loss_grad(s, y, v, logp.clone(), out=s)
    c = -torch.ones(4, dtype=torch.float64)
    src = torch.stack([grad[i] for i in rows])
    onehot = torch.zeros_like(p)
    onehot[torch.arange(4), y[rows].cpu()] = 1.0
    want = -(onehot - p)
    assert ((src.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2 * E[:, None] + 1e-30).all()
    assert float(grad[2].float().abs().max()) == 0.0


def test_more_than_a_million_short_rows(engine):
    n, m = 1_100_003, 5
    s, y = block(n, m, torch.float32, 11, masked=False)
    leaf = s.detach().requires_grad_(True)
    logp = engine.label_logprobs(leaf, y)
    (g,) = torch.autograd.grad(logp.sum(), leaf)
    l, p, e, E = formulas(s, y, 1.0)
    check_logp(logp, l, E, y)
    check_grad(g, s, y, 1.0, torch.ones(n).double(), torch.zeros(n).double(), p, e, E)
    loss, _ = engine.policy_loss(s, y, torch.ones(n, device="cuda"), logp.detach(), scale=1 / n)
    # r = exp(l - old) with old = l rounded: 1 to U |l|; minus the share of labelled rows, rounded
    assert abs(float(loss) + float((y >= 0).double().mean())) <= 1.01 * U * float(l.abs().max()) + 2 * U


def test_a_gradient_written_over_saved_scores_is_noticed(engine):
    s, y = block(6, 40, torch.float32, 4, masked=False)
    v = torch.ones(6, device="cuda")
    leaf = s.detach().requires_grad_(True)
    scores = leaf * 1.0
    logp = engine.label_logprobs(scores, y)  # its backward pass reads the scores
    engine.policy_loss_grad(scores, y, v, v, out=scores.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logp.sum().backward()
    with torch.inference_mode():  # no graph to protect
        t = s.clone()
        engine.policy_loss_grad(t, y, v, v, out=t)


@pytest.mark.parametrize("temperature", [1e-30, 1e30])
def test_the_largest_and_smallest_temperatures(engine, temperature):
    s, y = block(4, 40, torch.float32, 4, masked=True)
    logp = engine.label_logprobs(s, y, temperature)
    assert not torch.isnan(logp).any()
    if temperature > 1:  # uniform over the finite scores; |s| / 1e30 is below every rounding
        ref = torch.where(y.cpu() >= 0, -torch.isfinite(s.cpu()).sum(1).double().log(), 0.0)
        assert ((logp.cpu().double() - ref).abs() <= 44 * U + 2 * U * ref.abs()).all()
    else:  # the largest score alone
        best = s.gather(1, y.clamp(min=0)[:, None])[:, 0] == s.max(1).values
        assert ((logp == 0) == (best | (y < 0))).all()
