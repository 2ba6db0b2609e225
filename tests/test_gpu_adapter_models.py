"""GPU tests of a trained model with low-rank adapters (KgeModel.score_sp_adapted / score_po_adapted) and of the
losses on labels fed by it, against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import kge_oracle as K

pytestmark = pytest.mark.gpu

E, R, DIM, RANK, ADAPTERS, N = 203, 5, 32, 3, 4, 45


def make_model(name, base=None):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from kge import Config, Dataset, KgeModel

    torch.manual_seed(0)
    c = Config()
    c.set("model", name)
    c._import(name)
    if base:
        c.set(f"{name}.base_model.type", base)
        c._import(base)
    c.set("job.device", "cuda")
    c.set("dataset.num_entities", E)
    c.set("dataset.num_relations", R)
    c.set("lookup_embedder.dim", DIM)
    c.set("lookup_embedder.initialize", "normal_")
    c.set("lookup_embedder.initialize_args", {"mean": 0.0, "std": 1.0}, create=True)
    return KgeModel.create(c, Dataset(c, None))


def tables(model):
    ent, rel = model.get_s_embedder(), model.get_p_embedder()
    return [e._embeddings.weight.detach().double().cpu().numpy() for e in (ent, rel)]


def queries():
    g = torch.Generator().manual_seed(1)
    return (torch.randint(0, E, (N,), generator=g).cuda(), torch.randint(0, R, (N,), generator=g).cuda(),
            torch.randint(-1, ADAPTERS, (N,), generator=g).cuda())


def adapters_of(model, seed=2):
    mod = model.create_adapters(ADAPTERS, RANK, alpha=2.0)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        mod.b.copy_(torch.randn(mod.b.shape, generator=g))
    return mod


def adapted64(q, cand, mod, ids):
    """(scores, sum of the absolute products) in 64 bits."""
    a, b, s, ids = mod.a.detach().double().cpu(), mod.b.detach().double().cpu(), mod.scales.double().cpu(), ids.cpu()
    q, cand = torch.from_numpy(q), torch.from_numpy(np.ascontiguousarray(cand))
    y, size = q @ cand.t(), q.abs() @ cand.abs().t()
    for t in range(len(a)):
        i = (ids == t).nonzero()[:, 0]
        y[i] += s[t] * (q[i] @ a[t].t()) @ b[t].t()
        size[i] += s[t] * (q[i].abs() @ a[t].abs().t()) @ b[t].abs().t()
    return y, size


def query_size(name, prep, en, re):
    """The sum of the absolute products that make up each element of a query (en, re: absolute values).  Only ComplEx
    subtracts."""
    if name != "complex":
        return prep(en, re)
    (a, b), (c, d) = np.split(en, 2, 1), np.split(re, 2, 1)
    return np.concatenate([a * c + b * d, a * d + b * c], 1)


@pytest.mark.parametrize("direction", ["sp_", "_po"])
@pytest.mark.parametrize("name", ["complex", "distmult", "rescal", "cp", "simple"])
def test_scores_with_adapters(name, direction):
    """A query is a product or two per element (RESCAL: DIM), a score DIM products, h DIM and B h RANK: at most
    2 (2 DIM + RANK + 8) roundings of 2^-24 beside the sum of the absolute products, once with the query as it is and
    once with the absolute products that the query itself sums."""
    model = make_model(name)
    mod = adapters_of(model)
    e, p, ids = queries()
    ent, rel = tables(model)
    if direction == "sp_":
        got = model.score_sp_adapted(e, p, mod, ids)
        prep = lambda en, re: K.prep_sp(name, en, re)  # noqa: E731
    else:
        got = model.score_po_adapted(p, e, mod, ids)
        prep = lambda en, re: K.prep_po(name, re, en)  # noqa: E731
    en, re = ent[e.cpu().numpy()], rel[p.cpu().numpy()]
    q = prep(en, re)
    assert got.dtype == torch.float32 and got.shape == (N, E)
    want, size = adapted64(q, K.window(name, direction, ent), mod, ids)
    steps = 2 * (2 * DIM + RANK + 8) * 2.0 ** -24
    qa = query_size(name, prep, np.abs(en), np.abs(re))
    _, qsize = adapted64(qa, np.abs(K.window(name, direction, ent)), mod, ids)
    assert ((got.double().cpu() - want).abs() <= steps * (size + qsize)).all()


def test_reciprocal_relations():
    model = make_model("reciprocal_relations_model", "distmult")
    mod = adapters_of(model)
    e, p, ids = queries()
    ent, rel = tables(model)
    assert rel.shape[0] == 2 * R
    q = K.prep_sp("distmult", ent[e.cpu().numpy()], rel[p.cpu().numpy() + R])
    want, size = adapted64(q, ent, mod, ids)
    got = model.score_po_adapted(p, e, mod, ids)
    assert ((got.double().cpu() - want).abs() <= 2 * (2 * DIM + RANK + 8) * 2.0 ** -24 * 2 * size).all()


def test_new_adapters_change_nothing_and_only_adapters_train():
    """A run of the operators as they are used: reference log-probabilities under the frozen model, a policy loss and a
    preference loss on adapted scores, an optimiser's step on the adapters; the model's tables stay as they were."""
    from kge import engine

    model = make_model("complex")
    before = [t.copy() for t in tables(model)]
    mod = model.create_adapters(ADAPTERS, RANK)
    s, p, ids = queries()
    none = torch.full_like(ids, -1)
    plain = model.score_sp_adapted(s, p, mod, none).detach()
    assert torch.equal(model.score_sp_adapted(s, p, mod, ids).detach(), plain)  # B = 0

    g = torch.Generator().manual_seed(3)
    labels = torch.randint(0, E, (N,), generator=g).cuda()
    adv = torch.randn(N, generator=g).cuda()
    ref = engine.label_logprobs(plain, labels)
    opt = torch.optim.SGD(mod.parameters(), lr=0.1)
    for step in range(3):
        scores = model.score_sp_adapted(s, p, mod, ids)
        now = engine.label_logprobs(scores, labels)
        if step == 0:
            assert torch.equal(now.detach(), ref)
        ptr = torch.arange(0, 41, 5, device="cuda")  # 8 sequences of 5 answers, 4 pairs
        pi = torch.stack([ref[i:i + 5].sum() for i in range(0, 40, 5)])
        policy, _ = engine.policy_loss(scores, labels, adv, ref, ref, kl=0.1, scale=1 / N)
        preference, _ = engine.preference_loss(scores[:40], labels[:40], ptr, pi, beta=0.2)
        loss = policy + preference
        opt.zero_grad()
        loss.backward()
        assert torch.isfinite(loss) and torch.isfinite(mod.a.grad).all() and torch.isfinite(mod.b.grad).all()
        assert (mod.b.grad != 0).any() and ((mod.a.grad != 0).any() == (step > 0))
        opt.step()
    assert all(e._embeddings.weight.grad is None for e in (model.get_s_embedder(), model.get_p_embedder()))
    assert all((a == b).all() for a, b in zip(before, tables(model)))


def test_gradients_of_adapters_through_the_model():
    """The same kernels on the same query rows: the same bits as the operator called with them."""
    from kge import _lib as L
    from kge import engine

    model = make_model("cp")
    mod = adapters_of(model)
    s, p, ids = queries()
    up = torch.randn(N, E, generator=torch.Generator().manual_seed(4)).cuda()
    got = torch.autograd.grad(model.score_sp_adapted(s, p, mod, ids), (mod.a, mod.b), up)
    ent, rel = (t.detach() for t in model._lookup_tables())
    q = L.prep_query(L.CP, L.DIR_SP, ent, s, rel, p, N, DIM, rel.shape[1])
    want = torch.autograd.grad(engine.adapted_projection(q, engine.window(L.CP, L.DIR_SP, ent), mod.a, mod.b, ids,
                                                         mod.scales), (mod.a, mod.b), up)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_no_queries():
    model = make_model("distmult")
    mod = adapters_of(model)
    empty = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert model.score_sp_adapted(empty, empty, mod, empty).shape == (0, E)
