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


def _without_lost_weights(c):
    """tolerances for weights below 2^-125, which an fp32 exponential may flush to zero: all of what each contributes"""
    ref = oc.attention_reference(c)
    see, pos = oc.attention_sees(c)
    extra = {n: np.zeros(x[1].shape) for n, x in ref.items()}
    d, tk, h, g = c["q"].shape[3], c["k"].shape[1], c["q"].shape[2], c["k"].shape[2]
    scale = 1 / np.sqrt(d) if c["scale"] is None else c["scale"]
    for n in range(len(see)):
        for m in range(h):
            q, do = (c[x][n, :, m].astype(np.float64) for x in ("q", "do"))
            k, v = (c[x][n, :, m // (h // g)].astype(np.float64) for x in "kv")
            s = q @ k.T * scale
            if c["cap"]:
                s = c["cap"] * np.tanh(s / c["cap"])
            if c["slopes"] is not None:
                s = s - c["slopes"][m].astype(np.float64) * np.abs(pos[n][:, None] - np.arange(tk))
            s = np.where(see[n], s, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            lost = np.where(p < 2.0 ** -125, p, 0)
            ds = lost * (np.abs(do) @ np.abs(v).T + np.abs((do * (p @ v)).sum(1, keepdims=True))) * scale
            extra["out"][n, :, m] = lost @ np.abs(v)
            extra["dq"][n, :, m] = ds @ np.abs(k)
            extra["dk"][n, :, m // (h // g)] += ds.T @ np.abs(q)
            extra["dv"][n, :, m // (h // g)] += lost.T @ np.abs(do)
    return {n: (x[0], x[1] + 2 * extra[n]) for n, x in ref.items()}


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


def _tc_and_fp32(c, **kw):
    for flags in (0, adb.devices.FLAG_SIMT_DOT):
        dev = adb.devices.B200(0, flags=flags)
        oc.attention_check(oc.attention_run(dev, c, **kw), c)
        dev.close()


@pytest.mark.parametrize("d,heads", [(64, 4), (128, 2), (80, 2)])
@pytest.mark.parametrize("ratio", [2.0 ** -10, 2.0 ** -20, 2.0 ** -50])
def test_documents_that_fill_tiles_of_their_own(no_floors, d, heads, ratio):
    """a document's results do not depend on the size of another document's tokens in the same row"""
    tokens = 1000
    docs = np.tile(np.arange(tokens) // 256, (1, 1))
    c = oc.attention_case(1, tokens, tokens, heads, heads // 2, d, seed=3, docs=docs)
    small = (docs[0] % 2).astype(bool)
    for n, f in (("q", 1 / ratio), ("k", ratio), ("v", ratio), ("do", ratio)):
        c[n][:, small] *= np.float32(f)
    _tc_and_fp32(c)


@pytest.mark.parametrize("d", [64, 128])
def test_queries_in_front_of_a_key_do_not_set_its_units(no_floors, d):
    """under the causal mask the first 512 tokens' large gradients do not reach the keys behind them"""
    c = oc.attention_case(1, 1024, 1024, 2, 2, d, seed=5)
    c["do"][:, :512] *= np.float32(2.0 ** 40)
    _tc_and_fp32(c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("few", [False, True])
def test_keys_of_little_weight(no_floors, d, few):
    """keys whose weight is 2^-60 everywhere: small gradients, not zero or rounded ones; with them alone in a tile, too"""
    c = oc.attention_case(1, 300, 300, 2, 2, d, seed=6, scale=1.0, causal=False)
    c["q"][..., 0], c["k"][..., 0] = 1.0, 0.0
    c["q"][..., 1:] *= np.float32(1 / np.sqrt(d))
    at = [7, 130, 200] if few else np.arange(128, 256)
    c["k"][:, at, :, 0] = np.float32(-60 * np.log(2))
    ref = oc.attention_reference(c)
    # a query's gradients are held in halves in units of the row's largest: its first element, which these keys alone
    # make up, is as exact as the row's others are
    ref["dq"] = ref["dq"][0], np.broadcast_to(ref["dq"][1].max(-1, keepdims=True), ref["dq"][0].shape)
    for flags in (0, adb.devices.FLAG_SIMT_DOT):
        dev = adb.devices.B200(0, flags=flags)
        for n, x in oc.attention_run(dev, c).items():
            oc.close(n, x, *ref[n])
        dev.close()


@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("ratio", [2.0 ** -9, 2.0 ** -12, 2.0 ** -20, 2.0 ** -40])
def test_documents_token_by_token_in_one_tile(no_floors, d, ratio):
    c = _side_by_side(d, ratio)
    _tc_and_fp32(c)


@pytest.mark.parametrize("kw", [dict(), dict(cap=4.0), dict(slopes=True, causal=False), dict(cap=4.0, slopes=True)])
@pytest.mark.parametrize("tq,tk,heads,d", [(700, 700, 2, 128), (130, 4000, 1, 64), (300, 300, 2, 96)])
def test_rows_of_every_size(no_floors, kw, tq, tk, heads, d):
    """values and output gradients whose rows differ by up to 2^60, in every mixture; the middle case shares a tile's walk
    between blocks.  A row's results are made of what it sees, the largest first."""
    c = oc.attention_case(1, tq, tk, heads, heads, d, seed=tq, **kw)
    rng = np.random.default_rng(11)
    for n in ("v", "do"):
        size = rng.uniform(-30, 30, c[n].shape[1])
        size[:200] = rng.uniform(-8, 0, 200)[:len(size[:200])]     # a tile of similar rows, one across the border, the rest mixed
        c[n] *= np.exp2(np.round(size)).astype(np.float32)[None, :, None, None]
    c["k"][:, ::7] *= np.float32(2.0 ** -14)
    c["q"][:, ::5] *= np.float32(2.0 ** -14)
    ref = _without_lost_weights(c)      # slopes of 1/2 over 4000 keys: weights down to e^-2000
    for flags in (0, adb.devices.FLAG_SIMT_DOT):
        dev = adb.devices.B200(0, flags=flags)
        for n, x in oc.attention_run(dev, c).items():
            oc.close(n, x, *ref[n])
        dev.close()


def test_rows_of_zeros_beside_others(no_floors):
    """rows of zeros neither set a tile's unit nor need one"""
    c = oc.attention_case(1, 260, 260, 2, 1, 64, seed=8)
    for n in ("q", "k", "v", "do"):
        c[n][:, 3::4] = 0
    _tc_and_fp32(c)
    c["do"][:], c["v"][:] = 0, 0
    _tc_and_fp32(c)


@pytest.mark.parametrize("d", [64, 128, 160])
@pytest.mark.parametrize("exponent", [-115, -105, 110, 117])
@pytest.mark.parametrize("mixed", [False, True])
def test_values_near_the_ends_of_the_range(no_floors, d, exponent, mixed):
    """finite values give finite results up to 2^117 times normal ones; `mixed`: among rows that are 2^-30 as large"""
    c = oc.attention_case(1, 200, 200, 2, 2, d, seed=12)
    if mixed and exponent > 0:
        c["v"][:, ::3] *= np.float32(2.0 ** -30)
    ref = oc.attention_reference(c)                  # for values of order one: out, dq and dk are linear in them
    c["v"] *= np.float32(2.0 ** exponent)
    for flags in (0, adb.devices.FLAG_SIMT_DOT):
        dev = adb.devices.B200(0, flags=flags)
        for n, x in oc.attention_run(dev, c).items():
            size = 1.0 if n == "dv" else 2.0 ** exponent
            # 200 terms of a few roundings each, which among the subnormals leave half of 2^-149, times a factor (q, k) below 8
            oc.close(n, x.astype(np.float64) / size, ref[n][0], ref[n][1] + 200 * 4 * 8 * 2.0 ** -150 / size)
        dev.close()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("exponent", [-110, -60, 60, 110])
def test_large_queries_against_small_keys(no_floors, d, exponent):
    """scores of order one out of operands at opposite ends of the range"""
    c = oc.attention_case(1, 200, 200, 2, 2, d, seed=13)
    ref = oc.attention_reference(c)
    c["q"] *= np.float32(2.0 ** exponent)
    c["k"] *= np.float32(2.0 ** -exponent)
    for flags in (0, adb.devices.FLAG_SIMT_DOT):
        dev = adb.devices.B200(0, flags=flags)
        for n, x in oc.attention_run(dev, c).items():
            size = {"dq": 2.0 ** -exponent, "dk": 2.0 ** exponent}.get(n, 1.0)
            oc.close(n, x.astype(np.float64) / size, ref[n][0], ref[n][1] + 200 * 4 * 8 * 2.0 ** -150 / size)
        dev.close()


@pytest.mark.parametrize("d", [64, 128])
def test_a_single_key_has_a_weight_of_exactly_one(d):
    """documents of one token each: the output is the value to the halves' 22 bits, as the one score is its own maximum"""
    c = oc.attention_case(1, 200, 200, 2, 2, d, seed=21, docs=np.arange(200)[None], scale=2.0)
    got = oc.attention_run(adb.devices.B200(0), c, grad=False)["out"]
    # hi + lo leave half of 2^-21 of a value and 2^-39 of its row's largest
    oc.close("out", got, c["v"], 2.0 ** -22 * np.abs(c["v"]) + 2.0 ** -39 * np.abs(c["v"]).max(-1, keepdims=True) + oc.U * np.abs(c["v"]))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mixed", [False, True])
def test_queries_of_zeros_have_scores_of_zero(d, mixed):
    """whatever the keys and the scale are: the product of their units is out of range, the scores are not"""
    c = oc.attention_case(1, 150, 150, 2, 2, d, seed=22, scale=1000.0)
    c["q"][:], c["k"] = 0, c["k"] * np.float32(2.0 ** 122)
    if mixed:
        c["do"][:, ::3] *= np.float32(2.0 ** -30)
    got = oc.attention_run(adb.devices.B200(0), c)
    ref = oc.attention_reference(dict(c, k=c["k"] * np.float32(2.0 ** -122), scale=1.0))
    for n in ("out", "dv"):
        oc.close(n, got[n], *ref[n])
    assert not got["dk"].any()
