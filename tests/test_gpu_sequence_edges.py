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


# ---------------------------------------------------------------------------------------------
# values up to the largest
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("size", [3.2e38, 1.0, 1e-30])
@pytest.mark.parametrize("rise", [0.0, 0.9, 20.0])
@pytest.mark.parametrize("Hq,D,slots", [(1, 64, 40), (4, 64, 700), (3, 3, 50), (2, 96, 2100), (1, 256, 300), (2, 130, 90)])
def test_steps_over_values_up_to_the_largest(nn_gpu, Hq, D, slots, rise, size):
    """An average of values is between them, whatever they are and however the scores rise along the cache (in steps, to
    the base two, of `rise`)."""
    nn = nn_gpu
    rng = np.random.default_rng(D)
    q = np.zeros((1, Hq, D), np.float32)
    q[..., 0] = 1.0
    k = np.zeros((1, 1, slots + 1, D), np.float32)
    k[0, 0, :, 0] = (np.arange(slots + 1) * rise).astype(np.float32)
    v = (rng.uniform(0.5, 1.0, (1, 1, slots + 1, D)) * size).astype(np.float32)
    cache = nn.SinkCache(1, 1, slots + 1, 0, D)
    cache.k.set(k)
    cache.v.set(v)
    cache.set_lengths(slots)
    scale = float(np.float32(np.log(2.0)))
    y = nn.sink_attention_step(nn.Tensor_from_value(q), nn.Tensor_from_value(k[:, :, -1]), nn.Tensor_from_value(v[:, :, -1]), cache, scale=scale).np()
    x = k[0, 0, :, 0].astype(np.float64) * scale
    w = np.exp(x - x.max())
    want = np.einsum("n,nd->d", w / w.sum(), v[0, 0].astype(np.float64) / size)
    # a score of up to 2^11 * 20 is off by three roundings of it (times ln 2: less than one each), its weight by twice that and
    # by 2^-21; sums of n terms
    top = float(x.max())
    bound = 2 * 3 * U * min(top, 90 + 30) + 2.0 ** -21 + (slots + 8) * U + (6 * U * top if rise else 0)
    # (what is below the normal numbers: half of the smallest step for each term, times the power of two in front of the sum)
    base.close(y[0].astype(np.float64) / size, np.broadcast_to(want, (Hq, D)), bound + 2.0 ** -126 / size)


@pytest.mark.parametrize("S,D", [(40, 16), (64, 200), (150, 64), (300, 128)])
def test_attention_over_values_up_to_the_largest(nn_gpu, S, D):
    nn = nn_gpu
    rng = np.random.default_rng(D)
    q, k = (rng.standard_normal((1, 2, S, D)).astype(np.float32) for _ in range(2))
    v = rng.uniform(0.5, 1.0, (1, 2, S, D)).astype(np.float32)
    seen = base.visible(S, S, S, 0, (S,))
    want = base.plain_attention(*[torch.tensor(x, dtype=torch.float64) for x in (q, k, v)], seen, D ** -0.5).numpy()
    for size in (1.0, 2.0 ** 127, 2.0 ** -100):
        got = nn.sink_attention(*[nn.Tensor_from_value(x) for x in (q, k, v * np.float32(size))], S).np().astype(np.float64) / size
        # scores off by (D + 8) 2^-22 of their terms' magnitudes, weights by twice that and 2^-20, sums of S terms
        mag = float(np.einsum("bhtd,bhsd->bhts", np.abs(q), np.abs(k)).max()) * D ** -0.5
        base.close(got, want, 2 * (D + 8) * 2.0 ** -22 * mag + 2.0 ** -20 + (S + 8) * 2.0 ** -23)


# ---------------------------------------------------------------------------------------------
# what is not a number
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("S,D,window", [(30, 16, 9), (60, 64, 20), (300, 64, 40), (300, 128, 40), (100, 200, 30)])
@pytest.mark.parametrize("which", ["query", "key"])
@pytest.mark.parametrize("only_values", [False, True])
def test_what_is_not_a_number_reaches_the_gradients(nn_gpu, S, D, window, which, only_values):
    """A query row, or a key, of NaN: the gradients of what that query (all that see that key) sees are NaN, the others not."""
    nn = nn_gpu
    rng = np.random.default_rng(S + D)
    q, k, v, do = (rng.standard_normal((1, 2, S, D)).astype(np.float32) for _ in range(4))
    at = S // 2
    seen = base.visible(S, S, window, 0, (S,))[0, 0].numpy()
    if which == "query":
        q[:, 0, at, 0] = np.nan
        bad_rows = np.arange(S) == at
    else:
        k[:, 0, at, 0] = np.nan
        bad_rows = seen[:, at]
    bad_keys = seen[bad_rows].any(0)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    base.trainable(nn, *(t[2:] if only_values else t))
    y = nn.sink_attention(*t, window)
    nn.backward({y: nn.Tensor_from_value(do)})
    got = {"o": (y.np(), bad_rows), "dv": (t[2].get_grad().np(), bad_keys)}
    if not only_values:
        got["dq"], got["dk"] = (t[0].get_grad().np(), bad_rows), (t[1].get_grad().np(), bad_keys)
    for name, (x, bad) in got.items():
        assert np.isfinite(x[0, 1]).all(), name
        assert np.isfinite(x[0, 0][~bad]).all(), name
        assert np.isnan(x[0, 0][bad]).all(), name


# ---------------------------------------------------------------------------------------------
# scores far from zero
# ---------------------------------------------------------------------------------------------
SCORES = [1e3, 1e5, 1e6, 3e7, 1e8, 3e9, 1e12]
WINNERS = [(40, 16, 1), (300, 64, 2), (300, 128, 2), (140, 200, 1), (1500, 64, 1), (1200, 128, 1)]


def clear_winners(S, D, heads, score):
    """q, k, v, dO in which each query has one key far above all others, or two that are equal; the weights, and how far off
    they may be."""
    rng = np.random.default_rng(S + D)
    k = rng.choice([-1.0, 1.0], (heads, S, D)).astype(np.float32)
    k[:, 1::4] = k[:, 0:k[:, 1::4].shape[1] * 4:4]          # keys 4 n and 4 n + 1 are the same
    winner = np.array([[rng.integers(0, i + 1) for i in range(S)] for _ in range(heads)])
    q = (np.take_along_axis(k, winner[..., None], 1) * np.float32(score / D)).astype(np.float32)
    v, do = (rng.standard_normal((heads, S, D)).astype(np.float32) for _ in range(2))
    dots = np.einsum("hid,hjd->hij", q.astype(np.float64), k.astype(np.float64))
    dots[:, np.triu(np.ones((S, S), bool), 1)] = -np.inf
    w = np.exp(dots - dots.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    # Equal keys have equal scores.  A weight is off by 2^-20, and by what errors of the others' scores, (D + 8) 2^-22 of them, make
    # of their weights, which are `clear` at most.
    clear = float(np.sort(w, -1)[..., :-2].max())
    return q, k, v, do, w, 2.0 ** -20 + S * min(1.0, clear * np.exp(min(2 * (D + 8) * 2.0 ** -22 * score, 600.0)))


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("S,D,heads", WINNERS)
def test_clear_winners_at_any_score(nn_gpu, S, D, heads, score):
    """The weight of the winner is one, or a half each of two, however large the scores are."""
    nn = nn_gpu
    q, k, v, _, w, off = clear_winners(S, D, heads, score)
    got = nn.sink_attention(*[nn.Tensor_from_value(x[None]) for x in (q, k, v)], S, scale=1.0).np()[0]
    o = w @ v.astype(np.float64)
    base.close(got, o, off * np.abs(v).max() + 2.0 ** -21 * np.abs(o), "o")


@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("S,D,heads", WINNERS)
def test_gradients_of_clear_winners_at_any_score(nn_gpu, S, D, heads, score):
    nn = nn_gpu
    q, k, v, do, w, off = clear_winners(S, D, heads, score)
    t = [nn.Tensor_from_value(x[None]) for x in (q, k, v)]
    base.trainable(nn, *t)
    nn.backward({nn.sink_attention(*t, S, scale=1.0): nn.Tensor_from_value(do[None])})
    q, k, v, do = (x.astype(np.float64) for x in (q, k, v, do))
    ds = w * (np.einsum("hid,hjd->hij", do, v) - (do * (w @ v)).sum(-1, keepdims=True))
    want = {"dq": ds @ k, "dk": np.swapaxes(ds, 1, 2) @ q, "dv": np.swapaxes(w, 1, 2) @ do}
    got = dict(zip(("dq", "dk", "dv"), [x.get_grad().np()[0] for x in t]))
    # dP - delta: D products each, of (D + 8) 2^-22 of their magnitudes; dS is held as two fp16 numbers under a bound of 2^15 that is
    # at most 16 |dO| |V| (two powers of two, the sum of dP and delta, the largest of a head for a row's): what is below 2^-39 of
    # that is lost.
    mag = np.einsum("hid,hjd->hij", np.abs(do), np.abs(v))
    mag = mag + (w * mag).sum(-1, keepdims=True)
    lost = 2.0 ** -39 * 16 * np.linalg.norm(do, axis=-1).max() * np.linalg.norm(v, axis=-1).max()
    ds_off = (w * ((D + 8) * 2.0 ** -22) + off * (w > 1e-3)) * mag + 2.0 ** -21 * np.abs(ds) + lost
    base.close(got["dv"], want["dv"], (off + (S + 8) * U) * np.abs(do).sum(1, keepdims=True), "dv")
    base.close(got["dq"], want["dq"], ds_off @ np.abs(k), "dq")
    base.close(got["dk"], want["dk"], np.swapaxes(ds_off, 1, 2) @ np.abs(q), "dk")


@pytest.mark.parametrize("size_v,size_do", [(1e18, 1e14), (1e19, 1e2), (1e12, 1e8), (1.0, 1.0), (1e-18, 1e-8)])
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_through_small_weights(nn_gpu, D, size_v, size_do):
    """Keys whose weights are 10^-4 to 10^-10 in every row keep their gradients however large dO V is."""
    nn = nn_gpu
    S, scale = 200, 1.0
    rng = np.random.default_rng(D)
    q, k, v, do = (rng.standard_normal((1, 1, S, D)).astype(np.float32) for _ in range(4))
    q *= np.float32(0.05)
    q[..., 0] = 1.0
    k[..., 0] = 0.0
    k[:, :, 20:60, 0] = rng.uniform(-20.0, -8.0, 40)
    v, do = v * np.float32(size_v), do * np.float32(size_do)
    seen = base.visible(S, S, S, 0, (S,))
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = base.plain_attention(*r, seen, scale)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = base.attention_bounds(*[x.detach() for x in r], d64, seen, scale)
    # what is below 2^-39 of the bound of dS, at most 16 |dO| |V|, is lost (see above), and so are weights below 2^-39
    lost = 2.0 ** -39 * 16 * np.linalg.norm(do.astype(np.float64), axis=-1).max() * np.linalg.norm(v.astype(np.float64), axis=-1).max()
    rest = (2.0 ** -39 * np.abs(v).max() * S, lost * np.abs(k).sum(2, keepdims=True), lost * np.abs(q).sum(2, keepdims=True),
            2.0 ** -39 * np.abs(do).sum(2, keepdims=True))
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    base.trainable(nn, *t)
    y = nn.sink_attention(*t, S, scale=scale)
    nn.backward({y: nn.Tensor_from_value(do)})
    for name, g, w, b, c in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach()] + [x.grad for x in r], bounds,
                                rest):
        base.close(g.np(), w.numpy(), b.detach().numpy() + c, name)


# ---------------------------------------------------------------------------------------------
# gradients that are zero nearly everywhere
# ---------------------------------------------------------------------------------------------
def sparse_rows(S, where):
    rows = np.zeros(S, bool)
    if where == "last":
        rows[S - 20:] = True                                  # the loss is on the answer
    elif where == "turns":
        rows[S // 3:S // 3 + 9] = True
    else:
        rows[S // 2 + 1] = True
    return rows


@pytest.mark.parametrize("where", ["last", "turns", "one"])
@pytest.mark.parametrize("S,D", [(300, 64), (1000, 128), (900, 40)])
def test_gradient_of_some_rows(nn_gpu, S, D, where):
    nn = nn_gpu
    case = (1, 4, 2, S, S, D, S // 2, 4, None)
    (q, k, v, do), lens = base.attention_inputs(case)
    do[:, :, ~sparse_rows(S, where)] = 0.0
    do *= np.float32(3e-4)
    seen, scale = base.visible(S, S, S // 2, 4, lens), D ** -0.5
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = base.plain_attention(*r, seen, scale)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = base.attention_bounds(*[x.detach() for x in r], d64, seen, scale)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    base.trainable(nn, *t)
    y = nn.sink_attention(*t, S // 2, 4)
    nn.backward({y: nn.Tensor_from_value(do)})
    for name, g, w, b in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach()] + [x.grad for x in r], bounds):
        g = g.np()
        base.close(g, w.numpy(), b.detach().numpy() + 1e-30, name)
        norm = float(w.norm())
        assert np.linalg.norm(g - w.numpy()) <= 1e-5 * norm + bounds[4].get(name, 0.0) + 1e-30, name


@pytest.mark.parametrize("where", ["last", "turns", "one"])
def test_gradient_of_some_rows_stays_on_the_tensor_cores(nn_gpu, where):
    """The device time of the gradients with dO of zeros but in some rows, against that of a dense dO (the FP32 pipe takes ten
    times as long and more)."""
    nn = nn_gpu
    from litenn_b200 import _lib
    S, H, D = 4096, 8, 128
    rng = np.random.default_rng(2)
    t = [nn.Tensor_from_value(rng.standard_normal((1, H, S, D)).astype(np.float32)) for _ in range(3)]
    do = rng.standard_normal((1, H, S, D)).astype(np.float32)
    some = np.where(sparse_rows(S, where)[None, None, :, None], do, np.float32(0))
    opt = base.trainable(nn, *t)

    lib, dev = _lib.get_lib(), nn.devices.get_current()[0].index
    ev, ms = [ctypes.c_uint64(), ctypes.c_uint64()], ctypes.c_float()
    for e in ev:
        lib.lnn_event_create(dev, ctypes.byref(e))

    def pass_time(do_t):
        times = []
        for _ in range(4):
            opt.zero_grad()
            y = nn.sink_attention(*t, S)
            nn.devices.wait()
            lib.lnn_event_record(dev, ev[0].value)
            nn.backward({y: do_t})
            lib.lnn_event_record(dev, ev[1].value)
            nn.devices.wait()
            lib.lnn_event_elapsed_ms(dev, ev[0].value, ev[1].value, ctypes.byref(ms))
            times.append(ms.value)
        return min(times)

    dense, sparse = pass_time(nn.Tensor_from_value(do)), pass_time(nn.Tensor_from_value(some))
    for e in ev:
        lib.lnn_event_destroy(dev, e.value)
    assert sparse < 3 * dense, (sparse, dense)


@pytest.mark.parametrize("which", ["q", "k", "v", "k and do"])
@pytest.mark.parametrize("S,D,past", [(300, 64, 0), (700, 128, 100), (150, 40, 0)])
def test_operands_of_some_rows(nn_gpu, S, D, past, which):
    """Operands whose rows are zero but for a few between those that the guess of the scale looks at."""
    nn = nn_gpu
    case = (2, 4, 2, S - past, S, D, S // 2, 3, None)
    inputs, _ = base.attention_inputs(case)
    lens = (S, S - 40)
    for name, x in zip(("q", "k", "v", "do"), inputs):
        if name in which.split():
            keep = np.zeros(x.shape[2], bool)
            keep[x.shape[2] // 2 + 1:x.shape[2] // 2 + 3] = True
            x[:, :, ~keep] = 0.0
            x *= np.float32(700.0 if name == "do" else 2.0 ** -7)
    q, k, v, do = inputs
    seen, scale = base.visible(S - past, S, S // 2, 3, lens), D ** -0.5
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = base.plain_attention(*r, seen, scale)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = base.attention_bounds(*[x.detach() for x in r], d64, seen, scale)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    base.trainable(nn, *t)
    y = nn.sink_attention(*t, S // 2, 3, lengths_t=nn.Tensor_from_value(np.array(lens, np.float32)))
    nn.backward({y: nn.Tensor_from_value(do)})
    for name, g, w, b in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach()] + [x.grad for x in r], bounds):
        base.close(g.np(), w.numpy(), b.detach().numpy() + 1e-30, name)


@pytest.mark.parametrize("S,D", [(40, 16), (300, 64), (100, 200)])
def test_a_scale_of_nothing_is_the_mean(nn_gpu, S, D):
    """All weights of a row are the same, whatever the products are, and nothing reaches q and k."""
    nn = nn_gpu
    rng = np.random.default_rng(S)
    q, k, v, do = (rng.standard_normal((1, 2, S, D)).astype(np.float32) for _ in range(4))
    k *= np.float32(1e3)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    base.trainable(nn, *t)
    y = nn.sink_attention(*t, 7, scale=0.0)
    nn.backward({y: nn.Tensor_from_value(do)})
    w = base.visible(S, S, 7, 0, (S,))[0, 0].numpy().astype(np.float64)
    w /= w.sum(-1, keepdims=True)
    off = 2.0 ** -20 + 16 * U
    base.close(y.np(), np.einsum("ij,bhjd->bhid", w, v.astype(np.float64)), off * np.abs(v).max(), "o")
    base.close(t[2].get_grad().np(), np.einsum("ij,bhid->bhjd", w, do.astype(np.float64)), off * 7 * np.abs(do).max(), "dv")
    assert not t[0].get_grad().np().any() and not t[1].get_grad().np().any()


# ---------------------------------------------------------------------------------------------
# borders between the kernels
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("case", [(2, 4, 2, S, S, D, w, 2, None) for D in (72, 128) for S in (32, 33, 64) for w in (10, 100)] +
                         [(2, 4, 2, S, S, D, 20, 2, None) for D in (16, 64) for S in (64, 65)] +
                         [(1, 2, 1, 1, S, 128, S, 0, None) for S in (32, 33)])
def test_attention_at_the_borders_of_its_kernels(nn_gpu, case):
    base.test_sink_attention(nn_gpu, case)
