"""The orthogonalised updates refuse a call before any part of it runs."""
import math
from types import SimpleNamespace

import pytest
import torch

from spilltune_amd import _lib, engine, lora, moe, muon


def _table(*sizes):
    return (_lib.MatrixBatch * len(sizes))(*[
        _lib.MatrixBatch(x=4096, out=8192, count=n, rows=r, cols=c) for n, r, c in sizes])


def _call(*sizes):
    _lib.call("st_orthogonalize", len(sizes), _table(*sizes), 1, 5, 3.4445, -4.775, 2.0315, 1e-7, 4096,
              1 << 60, None)


MANY = ((1 << 24) - 1, 1, 1 << 20)  # more workgroups than a launch numbers


# behind matrices of the same table, of tables of another class of ranks, of more than
# one table holds
@pytest.mark.parametrize("before", [[(1, 4, 8)], [(1, 64, 100), (1, 4, 4096)], [(1, 16, 4096)] * 50,
                                    [(2, 20, 300), (0, 4, 4), (1, 200, 300)]])
def test_a_table_behind_others(before):
    with pytest.raises(ValueError, match="too many"):
        _call(*before, MANY)
    assert _lib.query("st_orthogonalize_workspace_bytes", len(before) + 1, _table(*before, MANY)) == -1
    assert _lib.query("st_orthogonalize_workspace_bytes", len(before), _table(*before)) >= 0


def test_the_query_tells_refused_sizes():
    for sizes in ((1, 1025, 1025), (1, -1, 4), (1, 4, 1 << 30), (1 << 24, 4, 4)):
        assert _lib.query("st_orthogonalize_workspace_bytes", 1, _table(sizes)) == -1


@pytest.mark.parametrize("sizes", [((1 << 22), 17, 20), ((1 << 22), 4, 2100), ((1 << 20), 33, 40)])
def test_many_small_matrices_are_taken(sizes):
    """Only the launches that are made bound the matrices of a call."""
    assert _lib.query("st_orthogonalize_workspace_bytes", 1, _table(sizes)) > 0


@pytest.mark.parametrize("kw,match", [
    ({"steps": 13}, "steps"), ({"steps": 0}, "steps"), ({"steps": 65, "coefficients": (1, 0, 0)}, "steps"),
    ({"steps": 5.0}, "integer"), ({"steps": True}, "integer"),
    ({"coefficients": (math.nan, 0.0, 0.0)}, "finite"), ({"coefficients": (1e3, 0.0, 0.0)}, "steps")])
def test_the_optimizer_refuses_its_rule_at_once(kw, match):
    with pytest.raises(ValueError, match=match):
        muon.Muon(**kw)
    assert muon.Muon(coefficients=iter((1, 0.5, 0))).coefficients == (1, 0.5, 0)


def _projection(rank, inner, outer):
    A, B = torch.rand(rank, inner), torch.rand(outer, rank)
    z = [t.clone() for t in (A, B, A, A, B, B)]
    return lora.LoRAProjection("p", rank, 8.0, inner, outer, A, B, *z)


def _state(projections):
    return [t.clone() for p in projections.values()
            for t in ((p.A, p.B, p.m_A, p.m_B) if hasattr(p, "A") else (p.weight, p.m, p.v))]


@pytest.mark.parametrize("last", [
    lambda: _projection(4, 8, 8),  # on the host, where nothing is orthogonalised
    lambda: _projection(1025, 1030, 1040),
    lambda: moe.make_expert_lora("e", 3, 1030, 1040, rank=1026, alpha=1.0, device="cpu")])
def test_a_refused_step_changes_nothing(last):
    t = torch.rand(5, 8)
    projections = {"embedding": SimpleNamespace(weight=t.clone(), grad=t + 1, m=t * 0, v=t * 0),
                   "first": _projection(4, 8, 16), "last": last()}
    optimizer = muon.Muon(lr=0.1, weight_decay=0.1, table=engine.AdamW(lr=0.1, weight_decay=0.1))
    before = _state(projections)
    for rule in ({}, {"steps": 20}, {"coefficients": (9.0, math.inf, 0.0)}):
        vars(optimizer).update(rule)
        with pytest.raises(ValueError, match="unsupported_capability"):
            optimizer.step(projections)
        assert all(torch.equal(a, b) for a, b in zip(before, _state(projections)))
        assert optimizer.step_count == 0 and optimizer.table.step_count == 0
