"""Programs with the transformer operators on the GPU against the oracle, and several handles of one GPU at once."""
import importlib
import threading

import numpy as np
import pytest

import operator_cases as oc
import operator_programs
from helpers import b200, oracle

pytestmark = pytest.mark.gpu
adb = importlib.import_module("autodiff-ir-rust_b200")
ad, ir = adb.autodiff, adb.ir


@pytest.mark.parametrize("chunk", range(4))
def test_random_operator_programs(chunk):
    """results over operands and views of them, in-place updates, branches and loops; the second execute replays a graph"""
    refused = ran = 0
    for seed in range(chunk * 25, chunk * 25 + 25):
        prog = operator_programs.build(seed)
        want = prog(oracle())
        tol = operator_programs.tolerance(want)
        if tol is None:
            continue
        try:
            runs = [prog(b200()), prog(b200())]
        except adb.devices.AdbError as e:
            assert "is a view when control flow joins" in str(e), str(e)
            refused += 1
            continue
        ran += 1
        for got in runs:
            for k in want:
                far = np.abs(np.asarray(got[k].data, np.float64) - np.asarray(want[k].data, np.float64)).max(initial=0)
                assert far <= tol[k], (seed, k, far, tol[k])
    assert ran >= 10, (ran, refused)


def test_handles_at_once_finish_and_agree():
    """programs on three handles of one GPU, executed by three threads at the same time: every iteration ends, without an
    error, with the bits of the first"""
    cases = [oc.attention_case(2, 400, 400, 4, 2, 64, seed=1), oc.attention_case(2, 300, 500, 4, 4, 128, seed=2, cap=5.0),
             oc.attention_case(3, 1, 3000, 8, 2, 128, seed=3, lengths=[3000, 17, 1200])]
    devs, blobs, ids, alive, first = [adb.devices.B200(0) for _ in cases], [], [], [], []
    for dev, c in zip(devs, cases):
        oc.start(dev)
        q, k, v = (oc.leaf(c[n]) for n in "qkv")
        out = ad.attention(q, k, v, cap=c["cap"], lengths=oc.data(c["lengths"]))
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
    wrong, done = [], [0] * len(cases)

    def work(i):
        try:
            for _ in range(30):
                devs[i].execute_blob(blobs[i])
                for n, t in ids[i].items():
                    assert np.array_equal(devs[i].get_tensor(t).numpy(), first[i][n]), n
                done[i] += 1
        except BaseException as e:
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not any(t.is_alive() for t in threads), done
    assert not wrong and done == [30] * len(cases), (wrong, done)
    for d in devs:
        d.close()
