"""Operators on tokens and sequences at the ends of their ranges: numbers that are none, values and scores far from one,
gradients that are zero nearly everywhere.  Against plain implementations in 64 bits; U is half a step of fp32."""
import ctypes

import numpy as np
import pytest
import torch

import test_gpu_sequence as base
from conftest import assert_bit_exact

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ---------------------------------------------------------------------------------------------
# numbers that are no token and no length
# ---------------------------------------------------------------------------------------------
def leave_in_the_pool(nn, shape, value):
    """The next tensor of this size gets memory that holds `value`."""
    nn.Tensor(shape).fill(value)


PRODUCTS = {
    # slot of the profile that counts the kernel, inputs, call
    "matmul": (0, [(700, 1030), (1030, 900)], lambda nn, a, b: nn.matmul(a, b)),
    "convolution": (1, [(2, 64, 32, 32), (64, 64, 3, 3)], lambda nn, a, b: nn.conv2D(a, b)),
    "strided convolution": (1, [(2, 64, 31, 31), (64, 64, 3, 3)], lambda nn, a, b: nn.conv2D(a, b, stride=2)),
    "few channels": (4, [(2, 3, 64, 64), (64, 3, 3, 3)], lambda nn, a, b: nn.conv2D(a, b)),
}


@pytest.mark.parametrize("which", list(PRODUCTS))
def test_products_behind_a_bad_token_number(nn_gpu, which):
    """A number that is no row counts as padding: what is queued behind it is computed all the same, and an update of
    weights too."""
    nn = nn_gpu
    from litenn_b200 import _lib
    lib, dev = _lib.get_lib(), nn.devices.get_current()[0].index
    slot, shapes, call = PRODUCTS[which]
    rng = np.random.default_rng(1)
    a, b = (rng.standard_normal(s).astype(np.float32) for s in shapes)
    a_t, b_t = nn.Tensor_from_value(a), nn.Tensor_from_value(b)
    opt = nn.optimizer.SGD([b_t], lr=0.01)
    ids_t, table_t = nn.Tensor_from_value(np.array([1, 7], np.float32)), nn.Tensor_from_value(np.ones((7, 4), np.float32))

    def step():
        y = call(nn, a_t, b_t)
        shape = tuple(y.shape)
        y.backward()
        opt.step()
        return y, shape

    y, shape = step()
    want, after = y.np(), b_t.np()
    launches, ms = ctypes.c_uint64(), ctypes.c_float()
    b_t.set(b)
    opt.zero_grad()
    del y
    for s in [shape] * 3 + shapes * 3:
        leave_in_the_pool(nn, s, float("nan"))
    lib.lnn_profile_enable(dev, 1)
    lib.lnn_profile_read(dev, slot, ctypes.byref(launches), ctypes.byref(ms))
    rows = nn.embedding(ids_t, table_t)
    y, _ = step()
    with pytest.raises(nn.LnnError, match="token number of an embedding"):
        rows.np()
    lib.lnn_profile_read(dev, slot, ctypes.byref(launches), ctypes.byref(ms))
    lib.lnn_profile_enable(dev, 0)
    assert launches.value > 0, "the tile engine was to be reached"
    assert_bit_exact(y.np(), want, "result")
    assert_bit_exact(b_t.np(), after, "weights after the step")
    nn.devices.wait()


def test_a_readback_reports_bad_numbers(nn_gpu):
    """Results that are read on the stream of their own come with the same report as those of np()."""
    nn = nn_gpu
    from litenn_b200 import _lib
    lib, dev = _lib.get_lib(), nn.devices.get_current()[0].index
    ids_t, table_t = nn.Tensor_from_value(np.array([1, 7], np.float32)), nn.Tensor_from_value(np.ones((7, 4), np.float32))
    good = nn.Tensor_from_value(np.array([1, 6], np.float32))
    host = ctypes.c_void_p()
    lib.lnn_host_alloc(32, ctypes.byref(host))
    try:
        for _ in range(2):
            y = nn.embedding(ids_t, table_t)
            lib.lnn_d2h_readback(dev, host, y._ptr(0), 32)
            with pytest.raises(nn.LnnError, match="token number of an embedding"):
                lib.lnn_wait_readback(dev)
            # reported once
            y = nn.embedding(good, table_t)
            lib.lnn_d2h_readback(dev, host, y._ptr(0), 32)
            lib.lnn_wait_readback(dev)
            assert list((ctypes.c_float * 8).from_address(host.value)) == [1.0] * 8
            assert (y.np() == 1).all()
        # a wait that expired, too (the word is written from the host)
        lib.lnn_debug_set_status(dev, _lib.E_TIMEOUT, 1, 7, 3)
        lib.lnn_d2h_readback(dev, host, y._ptr(0), 32)
        with pytest.raises(nn.LnnError, match="role 1, tile 7, step 3"):
            lib.lnn_wait_readback(dev)
        nn.devices.wait()
    finally:
        lib.lnn_host_free(host)
