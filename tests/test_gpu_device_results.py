"""Kept tensors that stay in HBM (FLAG_DEVICE_RESULTS): what can be had of them, and until when."""
import importlib

import numpy as np
import pytest

import operator_cases as oc

pytestmark = pytest.mark.gpu
adb = importlib.import_module("autodiff-ir-rust_b200")
ad, ir = adb.autodiff, adb.ir


@pytest.fixture()
def dev():
    d = adb.devices.B200(0, flags=adb.devices.FLAG_DEVICE_RESULTS)
    yield d
    d.close()


def _product(dev, n=256):
    """two kept tensors; the product runs on the tensor cores"""
    oc.start(dev)
    a = oc.leaf(np.eye(n) * 2)
    b = oc.leaf(np.arange(n * n).reshape(n, n) % 97)
    c = ad.dot(a, b)
    e = c + b
    for t in (c, e):
        t.forward().keep()
    ad.execute()
    return c.val().id, e.val().id, (np.arange(n * n) % 97).astype(np.float32)


def _more_than_fits(dev):
    """640 GB of results: the device's memory cannot be had, and the memory in use is given back before that shows"""
    oc.start(dev)
    x = oc.leaf(np.ones((1, 1))).broadcast(0, 400000).broadcast(1, 400000)
    (x * x).forward().keep()
    with pytest.raises(adb.devices.AdbError) as e:
        ad.execute()
    assert adb.devices.STATUS[e.value.status] == "ADB_ERR_OOM"


def test_results_are_gone_after_an_execute_that_found_no_memory(dev):
    c, e, b = _product(dev)
    assert np.array_equal(dev.get_tensor(c).numpy().reshape(-1), 2 * b)      # this one is on the host now
    _more_than_fits(dev)
    assert np.array_equal(dev.get_tensor(c).numpy().reshape(-1), 2 * b)
    assert dev.get_tensor(e).is_none
    assert dev.get_tensor_device(c) is None and dev.get_tensor_device(e) is None
    c, e, b = _product(dev)
    assert np.array_equal(dev.get_tensor(e).numpy().reshape(-1), 3 * b)


def test_results_are_gone_after_an_execute_that_failed_at_its_end(dev):
    _product(dev)
    dev.inject_dot_status(3)
    with pytest.raises(adb.devices.AdbError):
        c, e, b = _product(dev)
    for i in "abcdefghijklmnop":
        assert dev.get_tensor(i).is_none and dev.get_tensor_device(i) is None
    c, e, b = _product(dev)
    assert np.array_equal(dev.get_tensor(e).numpy().reshape(-1), 3 * b)


def test_host_copies_outlive_an_execute_that_found_no_memory():
    """without the flag every kept tensor is on the host when adb_execute returns"""
    d = adb.devices.B200(0)
    c, e, b = _product(d)
    _more_than_fits(d)
    assert np.array_equal(d.get_tensor(e).numpy().reshape(-1), 3 * b)
    assert d.get_tensor_device(e) is None
    d.close()


def test_a_kept_payload_of_the_callers_is_read_before_execute_returns(dev):
    """device payloads are borrowed for the duration of execute: a kept id that is bound to one holds what was there then"""
    torch = pytest.importorskip("torch")
    x = torch.arange(1000.0, device="cuda")
    torch.cuda.synchronize()
    oc.start(dev)
    a = ad.tensor(ir.DevicePayload(x.data_ptr(), x.numel(), x), [10, 100])
    y = a * 3.0
    a.forward().keep()
    y.forward().keep()
    ad.execute()
    x.fill_(-1.0)
    torch.cuda.synchronize()
    want = np.arange(1000, dtype=np.float32)
    assert np.array_equal(a.val().get().numpy().reshape(-1), want)
    assert np.array_equal(y.val().get().numpy().reshape(-1), 3 * want)
