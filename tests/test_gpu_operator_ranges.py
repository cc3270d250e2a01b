"""Attention where operands differ much in size: a result's error is bounded by what the result is made of, as fp32 sums
are, and not by rows that it does not see.  (`operator_cases.attention_reference` with its floors taken out.)"""
import importlib

import numpy as np
import pytest

import operator_cases as oc

pytestmark = pytest.mark.gpu
adb = importlib.import_module("autodiff-ir-rust_b200")


@pytest.fixture()
def no_floors(monkeypatch):
    monkeypatch.setattr(oc, "FLOOR_VALUE", 0.0)
    monkeypatch.setattr(oc, "FLOOR_WEIGHT", 0.0)


def _side_by_side(d, ratio, tokens=260):
    """two documents in turn, token by token; one has keys, values and output gradients `ratio` times the other's, and queries
    larger by as much, so that the scores of both are of order one"""
    docs = np.tile(np.arange(tokens) % 2, (2, 1))
    c = oc.attention_case(2, tokens, tokens, 4, 2, d, seed=7, docs=docs)
    for n, f in (("q", 1 / ratio), ("k", ratio), ("v", ratio), ("do", ratio)):
        c[n][:, 1::2] *= np.float32(f)
    return c


@pytest.mark.parametrize("d", [64, 128, 160])
@pytest.mark.parametrize("ratio", [2.0 ** -20, 2.0 ** -40])
def test_fp32_products_on_request(no_floors, d, ratio):
    """FLAG_SIMT_DOT: no halves anywhere"""
    c = _side_by_side(d, ratio)
    dev = adb.devices.B200(0, flags=adb.devices.FLAG_SIMT_DOT)
    oc.attention_check(oc.attention_run(dev, c), c)
    few = dict(c, **{n: c[n][:, -12:] for n in ("q", "do")})
    oc.attention_check(oc.attention_run(dev, few, grad=False), few)
    dev.close()
