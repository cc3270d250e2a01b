"""Transformer operators without a GPU: the oracle against the formulas in float64 and against differences, refusals by
the frontend and by the lowering, what the lowering makes of operands and results, and the data-parallel rule."""
import importlib
import struct
import threading

import numpy as np
import pytest

import operator_cases as oc
from oracle.oracle import OracleDevice

adb = importlib.import_module("autodiff-ir-rust_b200")
ad, ir, nn = adb.autodiff, adb.ir, adb.nn

MASKS = [
    dict(),
    dict(causal=False),
    dict(cap=2.0, slopes=True),
    dict(docs=[[0, 0, 1, 1, 1, 2, -1], [3, 3, 3, 3, -1, -1, -1]]),
    dict(prefix=[3, np.nan]),
    dict(lengths=[5, 0]),
    dict(causal=False, slopes=True, docs=[[1, 1, 1, 0, 0, 0, 0], [-1] * 7]),
]


@pytest.mark.parametrize("masks", MASKS)
def test_oracle_attention(masks):
    c = oc.attention_case(2, 7, 7, 4, 2, 5, seed=1, **masks)
    oc.attention_check(oc.attention_run(OracleDevice(), c), c)


@pytest.mark.parametrize("tq,tk,kw", [(1, 1, {}), (1, 9, {}), (3, 9, {}), (9, 3, {}), (9, 3, dict(causal=False)), (2, 6, dict(lengths=[1, 6]))])
def test_oracle_attention_lengths(tq, tk, kw):
    c = oc.attention_case(2, tq, tk, 2, 1, 4, seed=2, **kw)
    oc.attention_check(oc.attention_run(OracleDevice(), c), c)


@pytest.mark.parametrize("residual", [True, False])
def test_oracle_norm(residual):
    x = oc.norm_case((3, 4, 10), residual=residual)
    oc.norm_check(oc.norm_run(OracleDevice(), x), x)


@pytest.mark.parametrize("kw", [dict(rot=8), dict(rot=6, interleaved=True, gain=1.3), dict(rot=4, offset=100000), dict(rot=8, stretch=4.0)])
def test_oracle_rotary(kw):
    rng = np.random.default_rng(0)
    x, dy = (rng.standard_normal((2, 5, 3, 8)).astype(np.float32) for _ in range(2))
    got, want = oc.rotary_run(OracleDevice(), x, dy, **kw), oc.rotary_reference(x, dy, **kw)
    for k in got:
        oc.close(k, got[k], *want[k])


def test_gradients_against_differences():
    """the formulas' gradients, which every other test compares with, against central differences of their forward"""
    rng = np.random.default_rng(5)
    for masks in MASKS:
        c = oc.attention_case(2, 7, 7, 4, 2, 5, seed=3, **masks)
        ref = oc.attention_reference(c)
        for name in ("q", "k", "v"):
            step = rng.standard_normal(c[name].shape)
            ends = []
            for e in (1e-5, -1e-5):
                moved = dict(c, **{name: c[name].astype(np.float64) + e * step})
                ends.append((oc.attention_reference(moved)["out"][0] * c["do"]).sum())
            got, want = (ends[0] - ends[1]) / 2e-5, (ref["d" + name][0] * step).sum()
            # second-order differences: h^2 of a third derivative of order 1e2, and 1e-16 of sums of order 1e2 over h
            assert abs(got - want) < 1e-7 * (1 + abs(want)) + 1e-8
    x = {k: v.astype(np.float64) for k, v in oc.norm_case((3, 7)).items()}
    ref = oc.norm_reference(x)
    for name, gname in (("x", "dx"), ("r", "dr"), ("g", "dg")):
        step = rng.standard_normal(x[name].shape)
        ends = []
        for e in (1e-5, -1e-5):
            moved = oc.norm_reference(dict(x, **{name: x[name] + e * step}))
            ends.append((moved["y"][0] * x["dy"] + moved["h"][0] * x["dh"]).sum())
        assert abs((ends[0] - ends[1]) / 2e-5 - (ref[gname][0] * step).sum()) < 1e-8


def _zeros(*dim):
    return ad.tensor(np.arange(max(1, int(np.prod(dim))), dtype=np.float32)[:int(np.prod(dim))], list(dim))


@pytest.mark.parametrize("make", [
    lambda: ad.attention(_zeros(2, 3, 4, 8), _zeros(2, 3, 3, 8), _zeros(2, 3, 3, 8)),           # heads 4 over 3
    lambda: ad.attention(_zeros(2, 3, 4, 8), _zeros(2, 3, 4, 8), _zeros(2, 4, 4, 8)),           # values of another length
    lambda: ad.attention(_zeros(2, 3, 4, 8), _zeros(1, 3, 4, 8), _zeros(1, 3, 4, 8)),           # another batch
    lambda: ad.attention(_zeros(3, 4, 8), _zeros(3, 4, 8), _zeros(3, 4, 8)),                    # three axes
    lambda: ad.attention(_zeros(1, 1, 1, 257), _zeros(1, 1, 1, 257), _zeros(1, 1, 1, 257)),     # head too large
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, slopes=_zeros(2)),
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, docs=_zeros(1, 2)),
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, prefix=_zeros(1), causal=False),
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, lengths=_zeros(2)),
    lambda: ad.attention(_zeros(1, 4, 1, 8), _zeros(1, 3, 1, 8), _zeros(1, 3, 1, 8), docs=_zeros(1, 3)),
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, cap=-1.0),
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, cap=float("inf")),
    lambda: ad.attention(*[_zeros(1, 3, 1, 8)] * 3, scale=float("nan")),
    lambda: ad.rms_norm(_zeros(2, 4), _zeros(3)),
    lambda: ad.rms_norm(_zeros(2, 4), _zeros(4), _zeros(4, 2)),
    lambda: ad.rms_norm(_zeros(2, 4), _zeros(4), eps=-1.0),
    lambda: ad.rms_norm(_zeros(2, 4), _zeros(4), eps=float("nan")),
    lambda: ad.rms_norm(_zeros(2, 0), _zeros(0)),
    lambda: ad.rotary(_zeros(2, 3, 4), _zeros(2, 2)),
    lambda: ad.rotary(_zeros(2, 3, 1, 4), _zeros(2, 3)),
    lambda: ad.rotary(_zeros(2, 3, 1, 4), _zeros(3, 2)),
    lambda: ad.rotary(_zeros(2, 3, 1, 4), _zeros(2, 2), positions=_zeros(2)),
    lambda: ad.rotary(_zeros(2, 3, 1, 4), _zeros(2, 2), positions=_zeros(3), offset=1),
    lambda: ad.rotary(_zeros(2, 3, 1, 4), _zeros(2, 2), offset=1 << 25),
    lambda: nn.Rotary(3),
    lambda: nn.Rotary(4, stretch=0.0),
    lambda: nn.Rotary(4, blend=(4, 1, 100)),
    lambda: nn.SelfAttention(10, 3),
])
def test_frontend_refuses(make):
    oc.start(OracleDevice())
    with pytest.raises(ValueError):
        make()


def _lower(cmds, kept):
    proc = ir.IRProcedure("main")
    for c in cmds:
        proc.push(c)
    return adb.devices.lower_check(proc, set(kept))


def _mat(id_, *dim):
    return ("CreateMat", np.arange(int(np.prod(dim)), dtype=np.float32), list(dim), id_)


Q, K = _mat("q", 1, 3, 2, 8), _mat("k", 1, 3, 1, 8)
NONE4 = [None] * 4


@pytest.mark.parametrize("cmds,why", [
    ([Q, K, ("Attention", ["q", "k", "q"] + NONE4, ["o", "l"], [1], [1.0, 0.0])], "values must have"),
    ([Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o", "l"], [2], [1.0, 0.0])], "flag"),
    ([Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o", "l"], [1], [float("nan"), 0.0])], "scale"),
    ([Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o", "l"], [1], [1.0, -2.0])], "cap"),
    ([Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o", "o"], [1], [1.0, 0.0])], "same id"),
    ([Q, K, ("Attention", ["q", "k", None] + NONE4, ["o", "l"], [1], [1.0, 0.0])], "out of range"),
    ([Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o"], [1], [1.0, 0.0])], "number of results"),
    ([Q, K, ("Attention", ["q", "k", "k"], ["o", "l"], [1], [1.0, 0.0])], "number of operands"),
    ([Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o", "l"], [], [1.0, 0.0])], "number of parameters"),
    ([Q, K, _mat("s", 3), ("Attention", ["q", "k", "k", "s"] + NONE4[1:], ["o", "l"], [1], [1.0, 0.0])], "slopes"),
    ([Q, K, _mat("p", 1), ("Attention", ["q", "k", "k", None, None, "p", None], ["o", "l"], [0], [1.0, 0.0])], "prefix"),
    ([Q, K, ("AttentionGrad", ["q", "k", "k"] + NONE4 + ["q", "q", "q"], ["o", "l", "m"], [1], [1.0, 0.0])], "wrong shape"),
    ([Q, _mat("g", 7), ("RmsNorm", ["q", "g", None], ["o", "h"], [], [1e-6])], "scale"),
    ([Q, _mat("g", 8), ("RmsNorm", ["q", "g", None], ["o", "h"], [], [-1.0])], "eps"),
    ([Q, _mat("g", 8), ("RmsNormGrad", ["q", "g", "g", None], ["o", "h"], [], [1e-6])], "shape"),
    ([Q, _mat("t", 2, 5), ("Rotary", ["q", "t", None], ["o"], [0, 0, 0], [1.0])], "turns"),
    ([Q, _mat("t", 2, 4), ("Rotary", ["q", "t", None], ["o"], [0, 3, 0], [1.0])], "flag"),
    ([Q, _mat("t", 2, 4), ("Rotary", ["q", "t", None], ["o"], [0, 0, 1 << 30], [1.0])], "2^24"),
    ([Q, _mat("t", 2, 4), _mat("p", 4), ("Rotary", ["q", "t", "p"], ["o"], [0, 0, 0], [1.0])], "positions"),
    ([Q, K, ("Attention", ["q", "k", "x"] + NONE4, ["o", "l"], [1], [1.0, 0.0])], "before it is defined"),
])
def test_lowering_refuses(cmds, why):
    with pytest.raises(adb.devices.AdbError, match=why.replace("^", r"\^")):
        _lower(cmds, ["o"])


def test_truncated_operator_is_refused():
    proc = ir.IRProcedure("main")
    for c in (Q, K, ("Attention", ["q", "k", "k"] + NONE4, ["o", "l"], [1], [1.0, 0.0])):
        proc.push(c)
    blob, _ = ir.serialize(proc, {"o"})
    import ctypes
    L = adb.devices.load_library()
    err = ctypes.create_string_buffer(1000)
    head = blob.rindex(struct.pack("<BB", 33, 7))
    for end in range(head, head + 60, 3):
        rc = L.adb_lower_check(blob[:end], end, None, 0, None, 0, None, err, len(err))
        assert rc == 2, end


def _steps(plan, name):
    return [l for l in plan.splitlines() if f" {name} " in l]


def test_operands_are_read_where_they_lie():
    """heads split off a projection by views, permuted batches and broadcast heads need no copies"""
    oc.start(OracleDevice())
    x = _zeros(2, 6, 24)
    q = x.view([2, 6, 3, 8])
    k = _zeros(6, 2, 3, 8).permute([1, 0, 2, 3])
    out = ad.attention(q, k, _zeros(2, 6, 1, 8).broadcast(2, 3))
    out.forward()
    plan = adb.devices.lower_check(ad.current_ir(), {out.val().id})
    assert len(_steps(plan, "attention")) == 1 and "elw" not in plan, plan


def test_only_what_is_needed_runs():
    x = oc.norm_case((4, 8))
    oc.start(OracleDevice())
    a, g = oc.leaf(x["x"]), oc.leaf(x["g"])
    y, h = ad.rms_norm(a, g, oc.data(x["r"]))
    loss = y * oc.data(x["dy"]) + h * oc.data(x["dh"])
    loss.forward()
    loss.backward()
    plan = adb.devices.lower_check(ad.current_ir(), {a.grad().id})
    assert len(_steps(plan, "rms_norm")) == 1 and len(_steps(plan, "rms_norm_grad")) == 1
    assert "-> - " in _steps(plan, "rms_norm")[0], "the normalised rows are not needed for the gradient"
    plan = adb.devices.lower_check(ad.current_ir(), {y.val().id})
    assert not _steps(plan, "rms_norm_grad")


def test_an_operator_used_twice_has_one_gradient_command():
    oc.start(OracleDevice())
    x = _zeros(2, 3, 1, 4)
    y = nn.Rotary(4).f(x)
    loss = y * y + y
    loss.forward()
    loss.backward()
    assert sum(c[0] == "Rotary" for c in ad.current_ir().main) == 2
    g = x.grad()
    g.keep()
    y.val().keep()
    ad.execute()
    turned = np.asarray(y.val().get().data, np.float64)
    rest = oc.rotary_reference(np.zeros((2, 3, 1, 4), np.float32), (2 * turned + 1).reshape(2, 3, 1, 4), 4)["dx"]
    oc.close("dx", np.asarray(g.get().data).reshape(2, 3, 1, 4), rest[0], rest[1] + 1e-6 * np.abs(turned).max())


def test_a_leaf_that_sums_gradients_in_place_does_not_change_an_operators():
    """x's gradient starts as the value that also goes to the operator, and is added to before the operator sends its own"""
    oc.start(OracleDevice())
    x = oc.leaf(np.ones((1, 2, 1, 4)))
    w = oc.leaf(np.full((1, 2, 1, 4), 2.0))
    y = nn.Rotary(4).f(w)
    loss = (x + y) + x * 3.0
    loss.forward()
    loss.backward()
    gx, gw = x.grad(), w.grad()
    gx.keep()
    gw.keep()
    ad.execute()
    assert np.array_equal(np.asarray(gx.get().data), np.full(8, 4.0, np.float32))
    want = oc.rotary_reference(np.ones((1, 2, 1, 4)), np.ones((1, 2, 1, 4)), 4)["dx"]
    oc.close("dw", np.asarray(gw.get().data).reshape(1, 2, 1, 4), *want)


@pytest.mark.parametrize("shape", [(0, 3, 2, 4), (2, 0, 2, 4)])
def test_nothing_to_do(shape):
    oc.start(OracleDevice())
    x, g = _zeros(*shape), _zeros(4)
    y = ad.rms_norm(x, g)
    y.forward()
    z = nn.Rotary(4).f(x)
    z.forward()
    o = ad.attention(x, x, x)
    o.forward()
    ids = {t.val().id for t in (y, z, o)}
    plan = adb.devices.lower_check(ad.current_ir(), ids)
    assert not any(_steps(plan, n) for n in ("rms_norm", "rotary", "attention"))


def test_no_keys_gives_zeros():
    oc.start(OracleDevice())
    q, k = _zeros(2, 3, 2, 4), _zeros(2, 0, 2, 4)
    o = ad.attention(q, k, k)
    o.forward()
    plan = adb.devices.lower_check(ad.current_ir(), {o.val().id})
    assert not _steps(plan, "attention")


def _layer(seed=0, batch=4, tokens=5, width=16, heads=4, kv_heads=2, **masks):
    """norm, projections, rotary positions, attention and the residual, with every gradient"""
    rng = np.random.default_rng(seed)
    x = oc.leaf(rng.standard_normal((batch, tokens, width)))
    before = oc.leaf(rng.standard_normal((batch, tokens, width)))
    norm = nn.ResidualRMS(width)
    att = nn.SelfAttention(width, heads, kv_heads, rotary=nn.Rotary(4), rng=rng, **masks)
    y, h = norm.f(x, before)
    out = h + att.f(y)
    loss = nn.mse_loss(out, oc.leaf(rng.standard_normal((batch, tokens, width))).val().to_node())
    loss.forward()
    loss.backward()
    kept = {"loss": loss.val(), "x": x.grad()}
    kept.update({f"p{i}": p.grad() for i, p in enumerate(norm.params() + att.params())})
    for v in kept.values():
        v.keep()
    return kept


def test_layer_is_split_over_the_batch():
    """two ranks over half the sequences each, against one over all"""
    dev = OracleDevice()
    oc.start(dev)
    kept = _layer()
    blob, alive = ir.serialize(ad.current_ir(), ad.ret_dep_list(), inline_limit=1 << 30)
    dev.execute_blob(blob)
    want = {n: np.asarray(dev.get_tensor(v.id).data) for n, v in kept.items()}
    meet = threading.Barrier(2)
    parts = [None, None]
    got = [None, None]

    def rank(r):
        def reduce(a):
            parts[r] = a.copy()
            meet.wait(60)
            total = parts[0] + parts[1]
            meet.wait(60)
            a[:] = total

        d = OracleDevice(allreduce=reduce)
        d.execute_blob(adb.devices.shard_ir(blob, r, 2, 4))
        got[r] = {n: np.asarray(d.get_tensor(v.id).data) for n, v in kept.items()}

    threads = [threading.Thread(target=rank, args=(r,)) for r in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    both = {n: np.concatenate([got[0][n], got[1][n]]) if n == "x" else got[1][n] for n in want}
    for n in want:
        # sums over the batch are cut in two: a few roundings of the largest element
        assert np.abs(both[n] - want[n]).max() <= 64 * oc.U * max(np.abs(want[n]).max(), 1e-6), n


def test_mixed_distribution_is_refused():
    oc.start(OracleDevice())
    q, k = _zeros(4, 3, 2, 4), _zeros(1, 3, 2, 4).broadcast(0, 4)
    o = ad.attention(q, k, _zeros(4, 3, 2, 4).permute([0, 1, 2, 3]))
    o.forward()
    blob, alive = ir.serialize(ad.current_ir(), {o.val().id})
    adb.devices.shard_ir(blob, 0, 2, 4)      # the broadcast along the batch is cut like the rest
    oc.start(OracleDevice())
    docs = _zeros(2, 4)
    y = nn.Rotary(4).f(_zeros(2, 4, 1, 4), positions=docs.permute([0, 1]))
    y.forward()
    x = _zeros(4, 2)
    z = ad.rms_norm(x.t(), _zeros(4))
    z.forward()
    blob, alive = ir.serialize(ad.current_ir(), {y.val().id, z.val().id})
    with pytest.raises(adb.devices.AdbError, match="rows"):
        adb.devices.shard_ir(blob, 0, 2, 4)


@pytest.mark.parametrize("offset,tokens,good", [((1 << 24) - 2, 3, True), ((1 << 24) - 2, 4, False), (1 << 24, 1, True), (1 << 24, 2, False),
                                                (-(1 << 24), 2, True), (-(1 << 24) - 1, 2, False)])
def test_positions_end_where_floats_are_whole_numbers(offset, tokens, good):
    """beyond 2^24 a position would round to a neighbour's"""
    oc.start(OracleDevice())
    x, t = _zeros(1, tokens, 1, 4), _mat("t", 2, 2)
    cmds = [_mat("x", 1, tokens, 1, 4), t, ("Rotary", ["x", "t", None], ["y"], [0, 0, offset], [1.0])]
    if good:
        ad.rotary(x, _zeros(2, 2), offset=offset)
        _lower(cmds, ["y"])
        return
    with pytest.raises(ValueError, match="24"):
        ad.rotary(x, _zeros(2, 2), offset=offset)
    with pytest.raises(adb.devices.AdbError, match="24"):
        _lower(cmds, ["y"])


def test_more_tokens_than_positions_are_refused():
    """2^24 + 2 tokens counted from 0: the last one's position is no float"""
    oc.start(OracleDevice())
    x = _zeros(1, 1, 1, 2).broadcast(1, (1 << 24) + 2)
    with pytest.raises(ValueError, match="24"):
        ad.rotary(x, _zeros(2, 1))


def test_a_backward_pass_that_raised_leaves_no_gradients_behind():
    class Bad(ad.Node):
        def __init__(self, t): self.t = t
        def forward(self): return self.t.forward()
        def backward(self, grad): raise RuntimeError("no gradient")
        def dim(self): return self.t.dim()
        def val(self): return self.t.val()

    dev = OracleDevice()
    oc.start(dev)
    w = oc.leaf(np.ones((1, 2, 1, 4)))
    y = nn.Rotary(4).f(w)
    loss = y + ad.Tensor(Bad(oc.leaf(np.ones((1, 2, 1, 4)))))
    loss.forward()
    with pytest.raises(RuntimeError):
        loss.backward()
    again = y * 3.0
    again.forward()
    again.backward()
    g = w.grad()
    g.keep()
    ad.execute()
    want = oc.rotary_reference(np.ones((1, 2, 1, 4)), np.full((1, 2, 1, 4), 3.0), 4)["dx"]
    oc.close("dw", np.asarray(g.get().data).reshape(1, 2, 1, 4), *want)
