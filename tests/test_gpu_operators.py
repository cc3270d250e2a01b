"""Transformer operators on the GPU against their formulas in float64: sizes, strides and masks where kernels go wrong,
and a layer made of them."""
import importlib

import numpy as np
import pytest

import operator_cases as oc
from helpers import b200, oracle

pytestmark = pytest.mark.gpu
adb = importlib.import_module("autodiff-ir-rust_b200")
ad, ir, nn = adb.autodiff, adb.ir, adb.nn


# ---------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 5), (1, 4096), (9, 128), (300, 130), (1000, 256), (77, 512), (2500, 1024), (33, 1028),
                                        (65, 2048), (40, 3001), (5, 8192), (300, 5003), (7, 16384), (3, 16385), (70, 20000)])
def test_norm(rows, width, residual):
    x = oc.norm_case((rows, width), seed=width, residual=residual)
    oc.norm_check(oc.norm_run(b200(), x), x)


def test_norm_of_a_strided_view_and_a_scalar_axis():
    rng = np.random.default_rng(0)
    x = oc.norm_case((6, 4, 8))
    wide = rng.standard_normal((6, 4, 24)).astype(np.float32)
    wide[:, :, 8:16] = x["x"]
    dev = b200()
    oc.start(dev)
    part = oc.leaf(wide).view([6, 4, 3, 8]).i(1, 2)
    y, h = ad.rms_norm(part, oc.leaf(x["g"]), oc.leaf(x["r"].transpose(1, 0, 2).copy()).permute([1, 0, 2]))
    got = oc.finish({"y": y.forward(), "h": h.forward()})
    ref = oc.norm_reference(x)
    for k in got:
        oc.close(k, got[k], *ref[k])


def test_norm_extremes():
    """rows of zeros, of the smallest normals, of values whose squares overflow, and one with an infinity"""
    x = oc.norm_case((5, 64), residual=False)
    x["x"][0] = 0
    x["x"][1] = 2e-38
    x["x"][2] = 1e30
    x["x"][3, 7] = np.inf
    got = oc.norm_run(b200(), x, grad=False)["y"]
    assert np.array_equal(got[0], np.zeros(64)) and np.isfinite(got[1]).all()
    assert np.array_equal(got[2], np.zeros(64))            # 1 / sqrt(inf)
    assert np.isnan(got[3, 7]) and not got[3, 8].any()     # inf * 0, and finite * 0
    oc.close("rest", got[4:], *(v[4:] for v in oc.norm_reference({k: v if v is None or k == "g" else np.where(np.isfinite(v) & (np.abs(v) < 1e20), v, 0) for k, v in x.items()})["y"]))


def test_same_bits_every_time():
    x = oc.norm_case((3000, 1000))
    a, b = oc.norm_run(b200(), x), oc.norm_run(b200(), x)
    c = oc.attention_case(2, 300, 300, 4, 2, 64, docs=np.repeat(np.arange(3), 100)[None].repeat(2, 0))
    p, q = oc.attention_run(b200(), c), oc.attention_run(b200(), c)
    for one, two in ((a, b), (p, q)):
        for k in one:
            assert np.array_equal(one[k], two[k]), k


# ---------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("shape,rot,kw", [
    ((1, 1, 1, 2), 2, {}), ((2, 300, 8, 128), 128, {}), ((2, 300, 8, 128), 128, dict(interleaved=True)),
    ((3, 77, 5, 96), 64, dict(interleaved=True, stretch=8.0)), ((1, 1000, 1, 80), 48, dict(gain=1.2)), ((2, 33, 3, 7), 6, {}),
    ((2, 33, 3, 7), 6, dict(interleaved=True)), ((1, 3, 40, 256), 256, dict(offset=16000000)), ((1, 2, 1, 9000), 8000, {}),
    ((5, 1, 64, 64), 4, dict(offset=-3))])
def test_rotary(shape, rot, kw):
    rng = np.random.default_rng(rot)
    x, dy = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    for positions in (None, rng.integers(0, 1 << 24, shape[1]), rng.integers(0, 1 << 20, shape[:2])):
        if positions is not None and "offset" in kw:
            continue
        p = None if positions is None else positions.astype(np.float32)
        got, want = oc.rotary_run(b200(), x, dy, rot, positions=p, **kw), oc.rotary_reference(x, dy, rot, positions=p, **kw)
        for k in got:
            oc.close(k, got[k], *want[k])


def test_rotary_blend():
    """slow pairs are stretched wholly, fast ones not at all"""
    turn = nn.Rotary(64, stretch=8.0, blend=(1, 32, 4096))
    plain = nn.Rotary(64)
    ratio = plain.table.astype(np.float64).sum(0) / turn.table.astype(np.float64).sum(0)
    assert np.allclose(ratio[:8], 1) and np.allclose(ratio[-6:], 8) and (np.diff(ratio) > -1e-12).all()


# ---------------------------------------------------------------------------------------------------- attention
def _docs(b, t, size, pad):
    d = (np.arange(t)[None] + np.arange(b)[:, None] * 7) // size
    return np.where(np.arange(t)[None] >= t - pad * np.arange(b)[:, None], -1, d)


SIZES = [(1, 1, 1, 1, 1, 1), (2, 64, 64, 2, 2, 64), (1, 65, 65, 3, 1, 40), (2, 127, 129, 4, 2, 128), (1, 200, 333, 2, 2, 80), (1, 50, 70, 2, 1, 160),
         (1, 33, 40, 2, 2, 256), (2, 130, 260, 4, 1, 6), (1, 513, 513, 2, 1, 96), (1, 300, 1000, 1, 1, 128),
         (2, 17, 300, 4, 2, 64), (1, 63, 64, 2, 2, 128), (1, 700, 1300, 2, 1, 64), (8, 260, 260, 8, 4, 64)]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("masks", ["full", "causal", "cap", "docs", "prefix", "lengths", "all"])
def test_attention(size, masks):
    b, tq, tk, h, g, d = size
    kw = {"full": dict(causal=False), "causal": {}, "cap": dict(cap=3.0, slopes=True, causal=False),
          "docs": dict(docs=_docs(b, tk, 50, 9)), "prefix": dict(prefix=([tk // 3 + 1, 0] * b)[:b]),
          "lengths": dict(lengths=([max(0, tk - 40), tk] * b)[:b]),
          "all": dict(cap=20.0, slopes=True, docs=_docs(b, tk, 90, 20), prefix=([10, tk + 5] * b)[:b], lengths=([tk - tk // 5, tk // 2] * b)[:b])}[masks]
    c = oc.attention_case(b, tq, tk, h, g, d, seed=tq + d, **kw)
    oc.attention_check(oc.attention_run(b200(), c), c)


@pytest.mark.parametrize("tq,tk,causal", [(1, 1, True), (300, 20, True), (300, 20, False), (1, 700, False), (129, 128, True)])
def test_attention_with_more_queries_than_keys(tq, tk, causal):
    """under the causal mask the first queries stand before the first key and see nothing"""
    c = oc.attention_case(2, tq, tk, 2, 2, 64, causal=causal)
    oc.attention_check(oc.attention_run(b200(), c), c)


@pytest.mark.parametrize("d", [64, 128, 160])
@pytest.mark.parametrize("tq", [1, 150])
def test_nothing_from_unreachable_rows(d, tq):
    """padding and the unused end of a cache hold NaN and infinities; a sequence may be all padding"""
    b, t = 3, 200
    docs = np.zeros((b, t))
    docs[0, 150:] = -1
    docs[1, :] = -1
    lengths = [t, t, 170]
    for kw in (dict(docs=docs), dict(lengths=lengths), dict(lengths=[0, 5, 170])):
        c = oc.attention_case(b, tq, t, 4, 2, d, **kw)
        see, _ = oc.attention_sees(c)
        hidden_k, hidden_q = ~see.any(1), ~see.any(2)
        used = oc.attention_sees(dict(c, causal=False))[0].any(1)   # hidden from every query by more than their order
        c["k"][~used] = np.nan
        c["v"][~used] = np.inf
        c["q"][hidden_q] = np.nan
        c["do"][hidden_q] = -np.inf
        got = oc.attention_run(b200(), c)
        oc.attention_check(got, c)
        assert not got["out"][hidden_q].any() and not got["dq"][hidden_q].any()
        assert not got["dk"][hidden_k].any() and not got["dv"][hidden_k].any()


def test_lowest_values_and_large_scores():
    """scores of +-3e4 and constant rows: no overflow, weights of exactly one or equal weights"""
    c = oc.attention_case(1, 130, 130, 2, 2, 64, scale=1.0)
    c["q"][:, ::2] *= 1e3
    c["k"][:, ::3] = 0
    c["q"][:, 5] = 0
    got = oc.attention_run(b200(), c, grad=False)
    oc.attention_check(got, c)


@pytest.mark.parametrize("magnitude", [1e-30, 1e-12, 1e6, 1e15])
def test_attention_magnitudes(magnitude):
    """values and gradients far from one, and rows of very different magnitude side by side"""
    c = oc.attention_case(1, 200, 200, 4, 2, 64, seed=4)
    c["v"] *= np.float32(magnitude)
    c["do"] *= np.float32(magnitude if magnitude < 1e10 else 1.0)
    c["do"][:, ::5] *= np.float32(1e-6)
    c["v"][:, 1::4] *= np.float32(1e-4)
    oc.attention_check(oc.attention_run(b200(), c), c)


def test_attention_reads_views():
    """projections split into heads by views, a permuted batch, one head broadcast over four"""
    c = oc.attention_case(3, 90, 90, 4, 4, 32)
    c["v"] = np.repeat(c["v"][:, :, :1], 4, 2)
    oc.start(b200())
    rng = np.random.default_rng(0)
    wide = rng.standard_normal((3, 90, 2, 4, 32)).astype(np.float32)
    wide[:, :, 1] = c["q"]
    q = oc.leaf(wide).i(1, 2)
    k = oc.leaf(c["k"].transpose(1, 0, 2, 3)).permute([1, 0, 2, 3])
    v = oc.leaf(c["v"][:, :, :1]).broadcast(2, 4)
    out = ad.attention(q, k, v)
    got = oc.finish({"out": out.forward()})
    oc.attention_check(got, c)


def test_gradient_of_a_broadcast_head():
    """one head of keys and values repeated by a broadcast: its gradient is the sum over the copies"""
    c = oc.attention_case(2, 70, 70, 4, 4, 32)
    for n in "kv":
        c[n] = np.repeat(c[n][:, :, :1], 4, 2)
    ref = oc.attention_reference(c)
    oc.start(b200())
    q, k, v = oc.leaf(c["q"]), oc.leaf(c["k"][:, :, :1]), oc.leaf(c["v"][:, :, :1])
    out = ad.attention(q, k.broadcast(2, 4), v.broadcast(2, 4))
    loss = out * oc.data(c["do"])
    loss.forward()
    loss.backward()
    got = oc.finish({"dq": q.grad(), "dk": k.grad(), "dv": v.grad()})
    oc.close("dq", got["dq"], *ref["dq"])
    for n in ("dk", "dv"):
        want, tol = (x.sum(2, keepdims=True) for x in ref[n])
        oc.close(n, got[n].reshape(want.shape), want, tol + 4 * oc.U * np.abs(ref[n][0]).sum(2, keepdims=True))


@pytest.mark.parametrize("b,tq,tk,h,g,d,kw", [
    (1, 1, 1, 1, 1, 64, {}), (3, 1, 1025, 8, 2, 64, dict(slopes=True)), (2, 1, 5000, 4, 4, 128, dict(lengths=[4097, 33])),
    (1, 1, 60001, 1, 1, 128, {}), (2, 2, 700, 8, 1, 96, dict(cap=5.0)), (2, 5, 3000, 6, 2, 40, dict(lengths=[3000, 2])),
    (1, 4, 999, 16, 2, 80, dict(prefix=[998])), (4, 1, 300, 12, 3, 130, dict(docs=_docs(4, 300, 70, 10))), (2, 1, 257, 32, 1, 256, {}),
    (1, 3, 2, 2, 1, 64, {}), (2, 1, 4000, 10, 5, 30, dict(causal=False, slopes=True)), (40, 1, 90, 8, 8, 64, dict(lengths=np.arange(40) * 2)),
    (2, 8, 2500, 4, 4, 128, dict(lengths=[2500, 1200])), (1, 16, 4100, 2, 2, 64, {})])
def test_few_queries_against_a_cache(b, tq, tk, h, g, d, kw):
    c = oc.attention_case(b, tq, tk, h, g, d, seed=tk, **kw)
    oc.attention_check(oc.attention_run(b200(), c, grad=False), c)


@pytest.mark.parametrize("tq,tk,h,g,d,kw", [(1, 64, 2, 1, 64, {}), (5, 700, 6, 2, 128, dict(cap=8.0)), (20, 300, 2, 2, 40, dict(slopes=True)),
                                            (1, 63, 2, 2, 64, {}), (3, 200, 4, 1, 130, dict(causal=False))])
def test_gradient_of_few_queries(tq, tk, h, g, d, kw):
    c = oc.attention_case(2, tq, tk, h, g, d, seed=tq, **kw)
    oc.attention_check(oc.attention_run(b200(), c), c)


def test_a_cache_beyond_two_to_the_31_bytes():
    """offsets into keys pass 2^31 bytes: the last sequence's rows are the ones that count"""
    torch = pytest.importorskip("torch")
    b, t, g, d = 3, 1 << 20, 1, 256      # 2^28 elements a sequence, 3 GiB in all
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(b, t, g, d, generator=gen, device="cuda") for _ in range(2))
    q = torch.randn(b, 1, 2, d, generator=gen, device="cuda")
    lengths = torch.tensor([5.0, 0.0, float(t)], device="cuda")
    torch.cuda.synchronize()
    oc.start(b200())
    one = [ad.tensor(ir.DevicePayload(x.data_ptr(), x.numel(), x), list(x.shape)) for x in (q, k, v, lengths)]
    out = ad.attention(*one[:3], lengths=one[3])
    got = oc.finish({"out": out.forward()})["out"]
    assert not got[1].any()
    s = (k[2, :, 0].double() @ q[2, 0].double().T) / 16
    p = torch.softmax(s, 0)
    want = (p.T @ v[2, :, 0].double()).cpu().numpy()
    size = (p.T @ v[2, :, 0].double().abs()).cpu().numpy()
    # scores of up to 6 of 256 terms: (256 + 16 + 24) u of sum |q k| / 16 <= 30; sums of 2^20 / 64 in turn at most
    oc.close("out", got[2, 0], want, size * (2 * (296 * 30 + 64) + 16384 / 16) * oc.U)
    del k, v


# ---------------------------------------------------------------------------------------------------- in programs
def _train(dev, steps):
    """a layer trained for some steps inside an IR loop"""
    rng = np.random.default_rng(3)
    oc.start(dev)
    b, t, w = 2, 40, 64
    x, target = (oc.leaf(rng.standard_normal((b, t, w))) for _ in range(2))
    norm = nn.ResidualRMS(w)
    att = nn.SelfAttention(w, 4, 2, rotary=nn.Rotary(16), rng=rng, cap=10.0)
    opt = nn.SGD(norm.params() + att.params(), 0.1)
    kept = {}

    def body(_):
        y, h = norm.f(x, target)
        loss = nn.mse_loss(h + att.f(y), target)
        loss.forward()
        loss.backward()
        kept["loss"] = loss.val()
        kept.update({f"g{i}": p.grad() for i, p in enumerate(opt.n)})
        opt.step()
        opt.zero_grad()
        x.reset_grad()
        target.reset_grad()

    if steps is None:
        body(None)
    else:
        ad.ir_for(range(0, steps), body)
    kept.update({f"p{i}": p.val() for i, p in enumerate(opt.n)})
    return oc.finish(kept)


@pytest.mark.parametrize("steps", [None, 3])
def test_layer_trains_like_the_oracle(steps):
    """norm, projections, rotary, attention and their gradients in one program, also as a replayed loop body"""
    want, got = _train(oracle(), steps), _train(b200(), steps)
    for n in want:
        # the layer's products are held to 3e-5 of their largest element; four follow one another, and steps add up
        assert np.abs(got[n] - want[n]).max() <= 4e-4 * (steps or 1) * np.abs(want[n]).max(), n


def test_eager_captured_and_replayed():
    """the first execute launches kernel by kernel, the second captures a graph, the third replays it; a program in
    between with other sizes uses the same memory"""
    c = oc.attention_case(2, 200, 200, 4, 2, 64, docs=_docs(2, 200, 60, 30))
    other = oc.attention_case(1, 500, 500, 2, 2, 128)
    dev = adb.devices.B200(0)
    oc.start(dev)
    q, k, v = (oc.leaf(c[n]) for n in "qkv")
    out = ad.attention(q, k, v, docs=oc.data(c["docs"]))
    loss = out * oc.data(c["do"])
    loss.forward()
    loss.backward()
    kept = [out.val(), q.grad(), k.grad(), v.grad()]
    for t in kept:
        t.keep()
    proc, deps = ad.current_ir(), ad.ret_dep_list()
    blob, alive = ir.serialize(proc, deps)
    runs, replays = [], 0
    for i in range(5):
        dev.execute_blob(blob)
        replays += dev.stats()["graph_replays"]
        runs.append([np.asarray(dev.get_tensor(t.id).data) for t in kept])
        if i == 3:
            oc.attention_check(oc.attention_run(dev, other), other)
    assert replays >= 2    # (the other program may have moved the memory, which drops the graph)
    for r in runs[1:]:
        for x, y in zip(runs[0], r):
            assert np.array_equal(x, y)
    dev.close()


@pytest.mark.parametrize("flags", ["FLAG_NO_FUSION", "FLAG_NO_GRAPHS", "FLAG_PROFILE", "FLAG_SERIAL_GRAPHS", "FLAG_DETERMINISTIC"])
def test_layer_under_flags(flags):
    dev = adb.devices.B200(0, flags=getattr(adb.devices, flags))
    got = _train(dev, 2)
    dev.close()
    want = _train(oracle(), 2)
    for n in want:
        assert np.abs(got[n] - want[n]).max() <= 8e-4 * np.abs(want[n]).max(), n


def test_two_handles_at_once():
    """two programs on two handles of one GPU, executed by two threads at the same time"""
    import threading
    cases = [oc.attention_case(2, 400, 400, 4, 2, 64, seed=1), oc.attention_case(2, 300, 500, 4, 4, 128, seed=2, cap=5.0)]
    devs = [adb.devices.B200(0) for _ in cases]
    blobs, ids, alive, first = [], [], [], []
    for dev, c in zip(devs, cases):
        oc.start(dev)
        q, k, v = (oc.leaf(c[n]) for n in "qkv")
        out = ad.attention(q, k, v, cap=c["cap"])
        loss = out * oc.data(c["do"])
        loss.forward()
        loss.backward()
        kept = dict(out=out.val(), dq=q.grad(), dk=k.grad(), dv=v.grad())
        for t in kept.values():
            t.keep()
        blob, keep = ir.serialize(ad.current_ir(), ad.ret_dep_list())
        blobs.append(blob)
        alive.append(keep)
        ids.append({n: t.id for n, t in kept.items()})
        dev.execute_blob(blob)
        first.append({n: dev.get_tensor(t).numpy() for n, t in ids[-1].items()})
        oc.attention_check(first[-1], c)
    wrong = []

    def work(i):
        for _ in range(30):
            devs[i].execute_blob(blobs[i])
            if any(not np.array_equal(devs[i].get_tensor(t).numpy(), first[i][n]) for n, t in ids[i].items()):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong
    for d in devs:
        d.close()


def test_a_decoding_loop():
    """a cache that grows by a token a step inside one program: lengths are data, the plan stays"""
    room, d = 200, 64
    c = oc.attention_case(2, 1, room, 4, 2, d, lengths=[100, 3])
    oc.start(b200())
    q, k, v = (oc.data(c[x]) for x in "qkv")
    total, length = ad.zeros([2, 1, 4, d]), ad.tensor(c["lengths"], [2])

    def step(_):
        nonlocal total, length
        total += ad.attention(q, k, v, lengths=length)
        total.forward()
        length += np.float32(1.0)
        length.forward()

    ad.ir_for(range(0, 5), step)
    got = oc.finish({"total": total.val(), "length": length.val()})
    want, tol = 0, 0
    for i in range(5):
        ref = oc.attention_reference(dict(c, lengths=c["lengths"] + i))["out"]
        want, tol = want + ref[0], tol + ref[1] + 8 * oc.U * np.abs(ref[0])
    assert list(got["length"]) == [105, 8]
    oc.close("total", got["total"], want, tol)


def test_results_left_on_the_device():
    torch = pytest.importorskip("torch")
    dev = adb.devices.B200(0, flags=adb.devices.FLAG_DEVICE_RESULTS)
    x = oc.norm_case((33, 70))
    got = oc.norm_run(dev, x)       # adb_get_tensor copies on demand
    oc.norm_check(got, x)
    assert dev.stats()["readback_ms"] < 1.0
    oc.start(dev)
    y = ad.rms_norm(oc.leaf(x["x"]), oc.leaf(x["g"]))
    y.forward().keep()
    ad.execute()
    address, shape = dev.get_tensor_device(y.val().id)
    assert shape == [33, 70]

    class View:
        __cuda_array_interface__ = dict(shape=tuple(shape), typestr="<f4", data=(address, False), version=2)

    there = torch.as_tensor(View(), device="cuda").cpu().numpy()
    assert np.array_equal(there, y.val().get().numpy()) and np.array_equal(there, y.val().get().numpy())
    dev.close()


def test_result_over_its_operand():
    """a result id that is also an operand's"""
    x = oc.norm_case((10, 32), residual=False)
    proc = ir.IRProcedure("main")
    proc.push(("CreateMat", x["x"].reshape(-1), [10, 32], "x"))
    proc.push(("CreateMat", x["g"], [32], "g"))
    proc.push(("RmsNorm", ["x", "g", None], ["x", "h"], [], [1e-6]))
    proc.push(("RmsNorm", ["x", "g", None], ["y", "x"], [], [1e-6]))
    for dev in (b200(), oracle()):
        dev.execute(proc, {"x", "y", "h"})
        h, n, y = (dev.get_tensor(i).numpy() for i in ("h", "x", "y"))
        assert np.array_equal(h, x["x"])
        ref = oc.norm_reference(x)
        oc.close("x", n, *ref["y"])
        again = oc.norm_reference(dict(x, x=n))
        oc.close("y", y, *again["y"])


@pytest.mark.parametrize("b,tq,tk,h,g,d,kw", [
    (3, 8, 900, 4, 4, 128, dict(lengths=[900, 5, 400])), (2, 16, 700, 3, 3, 64, dict(cap=6.0, slopes=True)), (2, 31, 300, 1, 1, 32, {}),
    (2, 8, 500, 8, 2, 32, dict(docs=_docs(2, 500, 90, 30))), (1, 63, 200, 2, 2, 16, dict(prefix=[30])), (2, 9, 333, 2, 2, 100, dict(causal=False)),
    (1, 9, 400, 2, 2, 128, {}), (2, 10, 300, 1, 1, 90, {})])
def test_from_8_queries_on(b, tq, tk, h, g, d, kw):
    """either side of the rule between tiles and rows; the last two: too many rows, and a head size that rows of 16 bytes do not fit"""
    c = oc.attention_case(b, tq, tk, h, g, d, seed=tq, **kw)
    oc.attention_check(oc.attention_run(b200(), c, grad=False), c)


def test_few_queries_of_operands_off_the_16_byte_grid():
    """keys and values that start 4 bytes behind a boundary: the tile takes them although rows would be preferred"""
    c = oc.attention_case(1, 8, 300, 2, 2, 64, seed=3)
    oc.start(b200())
    wide = {n: np.concatenate([np.zeros(c[n].shape[:3] + (1,), np.float32), c[n]], 3) for n in "kv"}
    k, v = (oc.leaf(wide[n]).r(range(1, 65), 3) for n in "kv")
    out = ad.attention(oc.leaf(c["q"]), k, v)
    got = oc.finish({"out": out.forward()})
    oc.attention_check(got, c)


@pytest.mark.parametrize("b,tq,tk,h,g,d,kw", [
    (2, 1, 1025, 8, 2, 62, dict(slopes=True)), (3, 1, 700, 4, 4, 126, dict(lengths=[700, 0, 65])), (1, 3, 64, 2, 1, 5, {}),
    (2, 7, 500, 6, 3, 99, dict(docs=_docs(2, 500, 120, 40), cap=3.0)), (1, 1, 9000, 2, 2, 30, dict(causal=False))])
def test_few_queries_of_odd_head_sizes(b, tq, tk, h, g, d, kw):
    c = oc.attention_case(b, tq, tk, h, g, d, seed=d, **kw)
    oc.attention_check(oc.attention_run(b200(), c, grad=False), c)
