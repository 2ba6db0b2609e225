"""GPU tests of the low-rank adapters beside a shared projection (kge/adapter.py, csrc/adapter.hip)
against their formulas in 64 bits.

Tolerances (u = 2^-24).  A sum of `len` products in fp32 is off by at most 2 len u sum |product| (one
rounding per product and one per addition; bf16 products are exact).  h (and u) carry that error into the
second product; meeting bf16 they are split into hi + lo, 2^-16 of their size.  Results are rounded once: half a
step of their type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def engine():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from kge import _lib, engine
    _lib.lib()
    return engine


def inputs(n, d, m, k, r, dtype, seed, ids="mixed", pad=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731

    def rows(count, cols):  # rows of a wider buffer that starts off an alignment boundary
        flat = torch.full((offset + count * (cols + pad) + 8,), 99.0, dtype=dtype)
        v = flat[offset:offset + count * (cols + pad)].view(count, cols + pad)[:, :cols]
        v.copy_(rn(count, cols))
        dev = flat.cuda()
        return dev[offset:offset + count * (cols + pad)].view(count, cols + pad)[:, :cols]

    t = dict(x=rows(n, d), w=rows(m, d), a=rn(k, r, d).cuda(), b=rn(k, m, r).cuda(),
             scales=(torch.rand(k, generator=g) + 0.5).cuda(), dy=rows(n, m))
    if ids == "mixed":
        i = torch.randint(-1, k, (n,), generator=g)
    elif ids == "skewed":  # most rows with one adapter, some adapters without rows
        i = torch.where(torch.rand(n, generator=g) < 0.8, k // 2, torch.randint(0, (k + 1) // 2, (n,), generator=g))
    elif ids == "none":
        i = torch.full((n,), -1)
    else:
        i = torch.full((n,), k - 1)
    return t, i.cuda()


def reference(t, ids, dtype):
    """{name: (value, bound)} of y, dx, da, db in 64 bits."""
    x, w, a, b, s, dy = (t[name].detach().cpu().double() for name in ("x", "w", "a", "b", "scales", "dy"))
    ids = ids.cpu()
    n, d = x.shape
    m, (k, r) = w.shape[0], a.shape[:2]
    half = torch.finfo(dtype).eps / 2
    cut = 2.0 ** -16 if dtype == torch.bfloat16 else 0.0
    tol = lambda length: 2 * (length + 4) * U  # noqa: E731
    y, ey = x @ w.t(), tol(d) * (x.abs() @ w.abs().t())
    dx, edx = dy @ w, tol(m) * (dy.abs() @ w.abs())
    da, eda, db, edb = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(b), torch.zeros_like(b)
    for q in range(k):
        i = (ids == q).nonzero()[:, 0]
        if not len(i):
            continue
        A, B = a[q], b[q]
        h, eh = s[q] * (x[i] @ A.t()), s[q] * tol(d) * (x[i].abs() @ A.abs().t())
        u, eu = s[q] * (dy[i] @ B), s[q] * tol(m) * (dy[i].abs() @ B.abs())
        y[i] += h @ B.t()
        ey[i] += (eh + cut * h.abs() + tol(r) * h.abs()) @ B.abs().t()
        dx[i] += u @ A
        edx[i] += (eu + cut * u.abs() + tol(r) * u.abs()) @ A.abs()
        da[q], eda[q] = u.t() @ x[i], (eu + tol(len(i)) * u.abs()).t() @ x[i].abs()
        db[q], edb[q] = dy[i].t() @ h, dy[i].abs().t() @ (eh + tol(len(i)) * h.abs())
    return {name: (v, e + 4 * U * v.abs() + half * (v.abs() + e) + 1e-37)
            for name, v, e in (("y", y, ey), ("dx", dx, edx), ("da", da, eda), ("db", db, edb))}


def check(got, want, what):
    v, tol = want
    assert got.shape == v.shape, (what, got.shape)
    err = (got.detach().cpu().double() - v).abs()
    assert (err <= tol).all(), (what, float((err - tol).max()), float(err.max()))


def run(engine, t, ids, which=("x", "a", "b")):
    leaf = {name: t[name].detach().requires_grad_(name in which) for name in ("x", "a", "b")}
    y = engine.adapted_projection(leaf["x"], t["w"], leaf["a"], leaf["b"], ids, t["scales"])
    grads = torch.autograd.grad(y, [leaf[name] for name in which], t["dy"]) if which else ()
    return {"y": y, **{"d" + name: g for name, g in zip(which, grads)}}


SIZES = [  # n, d, m, k, r, ids, row padding, storage offset
    (1, 1, 1, 1, 1, "all", 0, 0), (1, 64, 40, 3, 4, "mixed", 0, 0), (2, 33, 17, 2, 3, "mixed", 0, 1),
    (3, 512, 1000, 5, 16, "mixed", 0, 0), (16, 200, 300, 16, 8, "mixed", 8, 0), (17, 77, 129, 40, 5, "mixed", 3, 3),
    (40, 128, 256, 3, 64, "skewed", 0, 0), (64, 96, 130, 64, 16, "mixed", 0, 8), (100, 300, 70, 7, 100, "mixed", 0, 0),
    (129, 256, 257, 2, 1, "skewed", 0, 0), (300, 64, 128, 237, 8, "mixed", 0, 0), (257, 520, 384, 1, 24, "all", 0, 0),
    (130, 40, 50, 4, 16, "none", 0, 0), (1500, 48, 600, 6, 8, "skewed", 8, 0), (5000, 16, 24, 3, 4, "skewed", 0, 0),
    (70, 2100, 4100, 4, 16, "mixed", 4, 4), (20, 64, 14541, 3, 16, "mixed", 0, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, d, m, k, r, ids, pad, offset", SIZES)
def test_projection_and_gradients(engine, n, d, m, k, r, ids, pad, offset, dtype):
    t, i = inputs(n, d, m, k, r, dtype, n + d + m, ids, pad, offset)
    want = reference(t, i, dtype)
    got = run(engine, t, i)
    for name in ("y", "dx", "da", "db"):
        check(got[name], want[name], name)
        assert got[name].dtype == dtype
    # a run without a gradient takes the path for few requests where there are few: the same bound
    with torch.no_grad():
        y = engine.adapted_projection(t["x"], t["w"], t["a"], t["b"], i, t["scales"])
    check(y, want["y"], "y")
    # a second run gives the same bits
    again = run(engine, t, i, ("a", "b"))
    assert torch.equal(again["da"], got["da"]) and torch.equal(again["db"], got["db"])
    for q in range(k):  # an adapter without rows has a zero gradient
        if not (i == q).any():
            assert (got["da"][q] == 0).all() and (got["db"][q] == 0).all()


def test_no_scales_is_ones_and_no_rows(engine):
    t, i = inputs(30, 64, 50, 4, 8, torch.float32, 0)
    one = dict(t, scales=torch.ones(4, device="cuda"))
    assert torch.equal(run(engine, dict(t, scales=None), i)["y"], run(engine, one, i)["y"])
    t, i = inputs(0, 64, 50, 4, 8, torch.float32, 0)
    got = run(engine, t, i)
    assert got["y"].shape == (0, 50) and got["dx"].shape == (0, 64)
    assert (got["da"] == 0).all() and (got["db"] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [3, 16, 40, 300])
def test_a_diverged_adapter_reaches_its_own_rows_only(engine, n, dtype):
    t, i = inputs(n, 64, 100, 4, 8, dtype, 5, "mixed")
    i[:4] = torch.tensor([0, 1, 2, -1][:min(n, 4)], device="cuda")
    clean = run(engine, t, i)
    for value in (float("nan"), float("inf")):
        bad = dict(t, a=t["a"].clone(), b=t["b"].clone())
        bad["a"][1] = value
        bad["b"][1] = value
        got = run(engine, bad, i)
        others = i != 1
        assert torch.equal(got["y"][others], clean["y"][others])
        assert torch.equal(got["dx"][others], clean["dx"][others])
        assert not torch.isfinite(got["y"][~others]).any()
        keep = torch.tensor([0, 2, 3])
        assert torch.equal(got["da"][keep], clean["da"][keep]) and torch.equal(got["db"][keep], clean["db"][keep])
    # a request with NaN keeps to itself and to its adapter's gradient
    t["x"][0] = float("nan")
    got = run(engine, t, i)
    assert torch.equal(got["y"][1:], clean["y"][1:]) and torch.isnan(got["y"][0]).all()
    assert torch.equal(got["da"][1:], clean["da"][1:])


def test_ids_out_of_range_poison_their_row_only(engine, monkeypatch):
    from kge import _lib as L
    monkeypatch.setattr(L, "CHECK_INDEX", False)
    for n in (4, 200):
        t, i = inputs(n, 64, 100, 4, 8, torch.float32, 5)
        clean = run(engine, t, i)
        j = i.clone()
        j[0], j[2] = 4, -7
        got = run(engine, t, j)
        rest = torch.ones(n, dtype=torch.bool)
        rest[0] = rest[2] = False
        assert torch.equal(got["y"][rest], clean["y"][rest])
        assert torch.isnan(got["y"][0]).all() and torch.isnan(got["y"][2]).all()
        assert torch.isfinite(got["da"]).all() and torch.isfinite(got["db"]).all()


def test_rows_do_not_depend_on_the_rest_of_the_batch_order(engine):
    """A permuted batch gives permuted rows, bit for bit (each row's sums go over its own row only)."""
    t, i = inputs(300, 96, 200, 9, 8, torch.bfloat16, 8)
    y = run(engine, t, i, ())["y"]
    p = torch.randperm(300, generator=torch.Generator().manual_seed(1)).cuda()
    z = run(engine, dict(t, x=t["x"][p].contiguous()), i[p], ())["y"]
    assert torch.equal(z, y[p])


def test_arguments_that_need_a_copy(engine):
    t, i = inputs(40, 64, 50, 4, 8, torch.float32, 3)
    y = run(engine, t, i)
    other = dict(t, x=t["x"].t().contiguous().t(), w=t["w"].t().contiguous().t(),
                 a=t["a"].transpose(1, 2).contiguous().transpose(1, 2), b=t["b"].transpose(1, 2).contiguous().transpose(1, 2),
                 dy=t["dy"].t().contiguous().t())
    z = run(engine, other, i.int())
    assert all(torch.equal(y[name], z[name]) for name in y)
    # expanded requests and an expanded upstream gradient (a sum's): gradients of all rows collect
    leaf = t["x"][:1].clone().requires_grad_(True)
    out = engine.adapted_projection(leaf.expand(40, 64), t["w"], t["a"], t["b"], torch.zeros_like(i), t["scales"])
    (g,) = torch.autograd.grad(out.sum(), leaf)
    m = t["w"].double() + t["scales"][0].double() * t["b"][0].double() @ t["a"][0].double()
    want = 40 * m.sum(0)
    bound = 40 * (t["w"].double().abs().sum(0) + 2 * (t["b"][0].double().abs() @ t["a"][0].double().abs()).sum(0))
    assert ((g[0].double() - want).abs() <= 2 * (50 + 64 + 40 + 12) * U * bound).all()


def test_gradients_against_differences(engine):
    """The operator is bilinear in (a, b) and linear in x: central differences are exact but for rounding."""
    t, i = inputs(9, 24, 20, 3, 4, torch.float32, 2)
    got = run(engine, t, i)
    h = 2.0 ** -3
    for name in ("x", "a", "b"):
        flat = torch.randperm(t[name].numel(), generator=torch.Generator().manual_seed(1))[:12]
        for e in flat.tolist():
            v = []
            for sign in (1, -1):
                moved = t[name].clone()
                moved.view(-1)[e] += sign * h
                with torch.no_grad():
                    y = engine.adapted_projection(*[{**t, name: moved}[q] for q in ("x", "w", "a", "b")], i, t["scales"])
                v.append(float((y.double() * t["dy"].double()).sum()))
            diff = (v[0] - v[1]) / (2 * h)
            # 180 values of y up to ~60, each off by 2 (24 + 12) u of its absolute sum (<= 200), times |dy| <= 4
            assert abs(diff - float(got["d" + name].reshape(-1)[e])) <= 180 * 72 * U * 200 * 4 / h


@pytest.mark.parametrize("n, dtype", [(1, torch.bfloat16), (16, torch.float32), (200, torch.bfloat16)])
def test_recorded_in_a_graph(engine, n, dtype):
    """Forward and backward recorded once and replayed on new contents and ids, with eager work between;
    two recorded graphs do not share a workspace."""
    t, i = inputs(n, 96, 130, 5, 8, dtype, 1)

    def work():
        got = run(engine, t, i)
        return [got[name].detach() for name in ("y", "dx", "da", "db")]

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
    for seed in range(4):
        new, ids = inputs(n, 96, 130, 5, 8, dtype, 90 + seed)
        for name in t:
            t[name].copy_(new[name])
        i.copy_(ids)
        want = [v.clone() for v in work()]
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_two_streams_at_once(engine):
    data = [inputs(200, 96, 500, 5, 8, torch.bfloat16, s) for s in range(2)]
    want = [run(engine, *d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for d, st in zip(data, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(run(engine, *d))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(a[name], b[name]) for name in b)


def test_tables_past_32_bit_offsets(engine):
    """A bf16 table of more than 2^31 elements: the last rows are addressed in 64 bits."""
    n, d, m, r = 2, 1024, 2200003, 4
    w = torch.zeros(m, d, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(0)
    last = torch.randn(200, d, device="cuda", generator=g).bfloat16()
    w[-200:] = last
    x = torch.randn(n, d, device="cuda", generator=g).bfloat16()
    a = torch.randn(1, r, d, device="cuda", generator=g).bfloat16()
    b = torch.zeros(1, m, r, device="cuda", dtype=torch.bfloat16)
    b[0, -200:] = torch.randn(200, r, device="cuda", generator=g).bfloat16()
    ids = torch.tensor([0, -1], device="cuda")
    t = dict(x=x, w=last, a=a, b=b[:, -200:], scales=torch.ones(1), dy=torch.zeros(n, 200))
    y = engine.adapted_projection(x, w, a, b, ids)
    check(y[:, -200:], reference(t, ids, torch.bfloat16)["y"], "y")
    assert (y[:, :-200] == 0).all()


def test_post_training_run(engine):
    """The operators together, as they are used: adapted scores of frozen queries -> policy loss (in one
    call with its gradient) and preference loss -> gradients of the adapters, against the same chain in 64 bits."""
    n, d, m, k, r = 48, 32, 200, 4, 4
    t, i = inputs(n, d, m, k, r, torch.float32, 6)
    x, w, scales = t["x"] * 0.2, t["w"] * 0.3, t["scales"]
    a, b = (t["a"] * 0.1).requires_grad_(True), (t["b"] * 0.1).requires_grad_(True)
    y = torch.randint(0, m, (n,), generator=torch.Generator().manual_seed(1)).cuda()
    y[5] = -1
    with torch.no_grad():
        ref = engine.label_logprobs(x @ w.t(), y)
    adv = torch.randn(n, generator=torch.Generator().manual_seed(2)).cuda()
    ptr = torch.arange(0, n + 1, 2, device="cuda")

    s = engine.adapted_projection(x, w, a, b, i, scales)
    old = engine.label_logprobs(s.detach(), y) - 0.01
    loss, logp, grad = engine.policy_loss_grad(s, y, adv, old, ref, kl=0.1, scale=1.0 / n)
    s.backward(grad)
    fused = (a.grad.clone(), b.grad.clone())
    a.grad = b.grad = None
    s = engine.adapted_projection(x, w, a, b, i, scales)
    loss2 = engine.policy_loss(s, y, adv, old, ref, kl=0.1, scale=1.0 / n)[0]
    pref = engine.preference_loss(s, y, ptr, None, beta=0.2, scale=2.0 / n)[0]
    loss2.backward(retain_graph=True)
    # |gradients| are below 1 here and the two routes differ by a few roundings of each
    for p, q in zip((a.grad, b.grad), fused):
        assert ((p - q).abs() <= 1e-5 * (1 + q.abs())).all()
    pref.backward()

    A, B = (v.detach().cpu().double().requires_grad_(True) for v in (a, b))
    X, W, S, I, Y = x.cpu().double(), w.cpu().double(), scales.cpu().double(), i.cpu(), y.cpu()
    rows = X @ W.t()
    extra = torch.stack([S[q] * (B[q] @ (A[q] @ v)) if q >= 0 else torch.zeros(m, dtype=torch.float64)
                         for q, v in zip(I.tolist(), X)])
    full = rows + extra
    l = torch.log_softmax(full, 1).gather(1, Y.clamp(min=0)[:, None])[:, 0] * (Y >= 0)
    q, dd = torch.exp(l - old.cpu().double()), ref.cpu().double() - l
    ad = adv.cpu().double()
    want = ((-torch.minimum(q * ad, q.clamp(0.8, 1.2) * ad) + 0.1 * (torch.exp(dd) - dd - 1)) * (Y >= 0)).sum() / n
    seq = l.view(-1, 2).sum(1)  # answers of two rows, pairs of answers
    z = 0.2 * (seq[0::2] - seq[1::2])
    want_pref = -(torch.nn.functional.logsigmoid(z)).sum() * 2 / n
    ga, gb = torch.autograd.grad(want + want_pref, (A, B))
    assert abs(float(loss) - float(want.detach())) <= 1e-5
    assert abs(float(pref.detach()) - float(want_pref.detach())) <= 1e-5
    # the scores (|s| < 20) carry 2 (32 + 4) u |s|: 1e-4 of them through softmax slopes below 1 into gradients
    for p, g in ((a.grad, ga), (b.grad, gb)):
        assert float((p.cpu().double() - g).abs().max()) <= 1e-4 * max(1.0, float(g.abs().max()))


def test_masked_in_place_before_the_backward_pass(engine):
    """Known answers set to -inf in the result itself, whatever the alignment of its rows (m odd)."""
    t, ids = inputs(40, 16, 51, 4, 3, torch.float32, 5)
    a, b = (t[q].detach().requires_grad_(True) for q in ("a", "b"))
    hide = torch.rand(40, 51, generator=torch.Generator().manual_seed(1)).cuda() < 0.2
    y = engine.adapted_projection(t["x"], t["w"], a, b, ids, t["scales"])
    masked = engine.adapted_projection(t["x"], t["w"], a, b, ids, t["scales"]).masked_fill_(hide, -float("inf"))
    assert torch.equal(masked.detach(), y.detach().masked_fill(hide, -float("inf")))
    got = torch.autograd.grad(masked, (a, b), t["dy"])
    want = torch.autograd.grad(y, (a, b), t["dy"].masked_fill(hide, 0.0))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("n", [3, 40, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_infinite_request_gives_infinities_in_its_row(engine, n, dtype):
    """W x and B h of a row with one infinity and zeros beside it, B and W of one sign each: inf, not NaN."""
    d, m, r = 8, 24, 2
    x = torch.zeros(n, d, dtype=dtype, device="cuda")
    x[:, 0] = 1.0
    x[1, 0] = float("inf")
    w = torch.ones(m, d, dtype=dtype, device="cuda")
    a = torch.ones(2, r, d, dtype=dtype, device="cuda")
    b = torch.ones(2, m, r, dtype=dtype, device="cuda")
    ids = (torch.arange(n, device="cuda") % 2)
    y = engine.adapted_projection(x, w, a, b, ids)
    rest = torch.arange(n, device="cuda") != 1
    assert (y[1] == float("inf")).all() and (y[rest] == 3.0).all()


@pytest.mark.parametrize("n, d, m, k, r, ids", [
    (70001, 8, 12, 5, 2, "mixed"), (40000, 8, 8, 900, 1, "skewed"), (9000, 8, 9, 4100, 2, "mixed"),
    (50, 24, 20, 40000, 3, "mixed")])
def test_sorted_plan(engine, monkeypatch, n, d, m, k, r, ids):
    """Many rows or many adapters: the order comes from a radix sort (of one digit, of two from 2046 adapters on)."""
    t, i = inputs(n, d, m, k, r, torch.float32, n + k, ids)
    want = reference(t, i, torch.float32)
    got = run(engine, t, i)
    for name in ("y", "dx", "da", "db"):
        check(got[name], want[name], name)
    again = run(engine, t, i)
    assert all(torch.equal(again[name], got[name]) for name in got)
    from kge import _lib as L
    monkeypatch.setattr(L, "CHECK_INDEX", False)
    bad = i.clone()
    bad[1::7], bad[2::11] = k + 3, -5
    out = (bad < -1) | (bad >= k)
    y = run(engine, t, bad)["y"]
    assert torch.isnan(y[out]).all() and torch.equal(y[~out], got["y"][~out])


def test_gradients_beside_a_table_of_millions_of_rows(engine):
    n, d, m, k, r = 3, 4, 4_300_007, 2, 1
    t, i = inputs(n, d, m, k, r, torch.float32, 1, "all")
    want, got = reference(t, i, torch.float32), run(engine, t, i)
    for name in ("y", "dx", "da", "db"):
        check(got[name], want[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, d, m, k, r, ids", [
    (100, 40, 20001, 5, 4, "mixed"), (70, 9000, 130, 3, 16, "mixed"), (33, 4100, 4100, 2, 1, "all"),
    (200, 8192, 33, 4, 24, "none")])
def test_split_sums(engine, n, d, m, k, r, ids, dtype):
    """Few results of long sums: split over workgroups and joined, in dx (m long), forwards (d long) or both."""
    t, i = inputs(n, d, m, k, r, dtype, n + d, ids, 3, 1)
    want, got = reference(t, i, dtype), run(engine, t, i)
    for name in ("y", "dx", "da", "db"):
        check(got[name], want[name], name)
    again = run(engine, t, i)
    assert all(torch.equal(again[name], got[name]) for name in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, d, m, k, r, ids", [
    (66000, 16, 20, 7, 8, "mixed"), (700, 64, 64, 30, 16, "skewed"), (150, 65, 63, 40, 20, "mixed")])
def test_narrow_results(engine, n, d, m, k, r, ids, dtype):
    """At most 64 columns of y or dx, in tiles of 128 rows and of 64."""
    t, i = inputs(n, d, m, k, r, dtype, n + m, ids)
    want, got = reference(t, i, dtype), run(engine, t, i)
    for name in ("y", "dx", "da", "db"):
        check(got[name], want[name], name)


@pytest.mark.parametrize("n, d, m, k, r", [(60000, 16, 12, 500, 2), (50, 40, 20001, 5, 4), (40, 9000, 30, 3, 3)])
def test_sorted_plans_and_split_sums_recorded_in_a_graph(engine, n, d, m, k, r):
    t, i = inputs(n, d, m, k, r, torch.float32, 1)

    def work():
        got = run(engine, t, i)
        return [got[name].detach() for name in ("y", "dx", "da", "db")]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for seed in range(3):
        new, ids = inputs(n, d, m, k, r, torch.float32, 90 + seed, "skewed")
        for name in t:
            t[name].copy_(new[name])
        i.copy_(ids)
        want = [v.clone() for v in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_no_rows_beside_many_adapters(engine):
    t, i = inputs(0, 4, 5, 30000, 1, torch.float32, 0)
    got = run(engine, t, i)
    assert got["y"].shape == (0, 5) and (got["da"] == 0).all() and (got["db"] == 0).all()
