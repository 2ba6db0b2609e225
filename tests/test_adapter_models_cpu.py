"""Refusals of a model with low-rank adapters, reached on the CPU (no launch)."""
import pytest
import torch

from kge import Config, Dataset, KgeModel
from kge import _lib as L
from kge import engine


def make_model(name, dropout=0.0):
    c = Config()
    c.set("model", name)
    c._import(name)
    c.set("job.device", "cpu")
    c.set("dataset.num_entities", 7)
    c.set("dataset.num_relations", 2)
    c.set("lookup_embedder.dim", 8)
    c.set("lookup_embedder.dropout", dropout)
    return KgeModel.create(c, Dataset(c, None))


IDX = torch.tensor([0, 1])


@pytest.mark.parametrize("name", ["transe", "rotate"])
def test_distance_models_are_refused(name):
    model = make_model(name)
    for call in (lambda: model.create_adapters(2, 3), lambda: model.score_sp_adapted(IDX, IDX, None, IDX),
                 lambda: model.score_po_adapted(IDX, IDX, None, IDX)):
        with pytest.raises(ValueError, match="bilinear"):
            call()


def test_dropout_is_refused_while_training_only():
    model = make_model("complex", dropout=0.5)
    with pytest.raises(ValueError, match="dropout"):
        model.create_adapters(2, 3)
    model.eval()
    assert model.create_adapters(2, 3).a.shape == (2, 3, 8)


@pytest.mark.parametrize("name, width", [("complex", 8), ("cp", 4), ("distmult", 8)])
def test_width_follows_the_query(name, width):
    mod = make_model(name).create_adapters(3, 2, alpha=1.0)
    assert mod.a.shape == (3, 2, width) and mod.b.shape == (3, 7, 2) and (mod.scales == 0.5).all()


def test_arguments_refused():
    model = make_model("complex")
    mod = model.create_adapters(2, 3)
    with pytest.raises(ValueError, match="per query"):
        model.score_sp_adapted(IDX, IDX[:1], mod, IDX)
    with pytest.raises(L.EngineError, match="MI355X"):
        model.score_sp_adapted(IDX, IDX, mod, IDX)
    ent, rel = model._lookup_tables()
    with pytest.raises(ValueError, match="frozen"):
        engine.score_all_adapted(L.COMPLEX, L.DIR_SP, ent, IDX, rel.detach(), IDX, mod.a, mod.b, IDX)
    with pytest.raises(ValueError, match="bilinear"):
        engine.score_all_adapted(L.TRANSE, L.DIR_SP, ent, IDX, rel, IDX, mod.a, mod.b, IDX)
