"""Operators on tokens and sequences against plain implementations in 64 bits (torch on the CPU, gradients by its
autograd).  Tolerances follow from the number of roundings; U is half a step of fp32."""
import math

import numpy as np
import pytest
import torch

from conftest import assert_bit_exact

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def close(got, want, bound, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, f"{what}: {got.shape} != {want.shape}"
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    ok = (off <= bound) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok.all(), f"{what}: {int((~ok).sum())} of {ok.size} elements off, worst {np.nanmax(np.where(ok, 0, off))}"


def trainable(nn, *tensors):
    return nn.optimizer.SGD(list(tensors))


# ---------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------
def some_ids(rng, n, vocab, kind):
    if kind == "same":
        return np.full(n, vocab - 1, np.float32)
    if kind == "padded":
        return np.full(n, -1, np.float32)
    ids = np.minimum((np.exp(rng.random(n) * math.log(vocab)) - 1).astype(np.int64), vocab - 1).astype(np.float32)
    if kind == "mixed":
        ids[rng.random(n) < 0.2] = -1
    return ids


@pytest.mark.parametrize("n,vocab,dim,kind", [
    (1, 1, 1, "all"), (1, 7, 3, "all"), (1, 9, 4, "padded"), (31, 2, 4, "mixed"), (32, 1, 5, "same"), (33, 300, 8, "same"),
    (1000, 3, 17, "mixed"), (4097, 300, 64, "all"), (2500, 70000, 8, "mixed"), (700, 255, 1028, "mixed"),
    (513, 256, 4, "padded"), (5000, 5, 260, "same"), (70001, 3, 5, "same"), (16385, 50001, 12, "all"), (300, 1 << 24, 1, "mixed")])
def test_embedding(nn_gpu, n, vocab, dim, kind):
    nn = nn_gpu
    rng = np.random.default_rng(n + vocab)
    ids = some_ids(rng, n, vocab, kind)
    table, dy = rng.standard_normal((vocab, dim)).astype(np.float32), rng.standard_normal((n, dim)).astype(np.float32)
    ids_t, table_t, dy_t = (nn.Tensor_from_value(x) for x in (ids, table, dy))
    opt = trainable(nn, table_t)
    y = nn.embedding(ids_t, table_t, 1.7)
    at = ids.astype(np.int64)
    want = np.where((at >= 0)[:, None], table[at] * np.float32(1.7), np.float32(0))
    assert_bit_exact(y.np(), want, "rows")
    nn.backward({y: dy_t})
    got = table_t.get_grad().np()
    sums, size, count = np.zeros((vocab, dim)), np.zeros((vocab, dim)), np.zeros(vocab)
    real = at >= 0
    np.add.at(sums, at[real], dy[real].astype(np.float64))
    np.add.at(size, at[real], np.abs(dy[real]).astype(np.float64))
    np.add.at(count, at[real], 1)
    scale = float(np.float32(1.7))
    # n - 1 additions in some order and one product
    bound = (count[:, None] + 1) * U * size * scale
    close(got, sums * scale, bound, "gradient")
    # a second pass adds, and gives the same bits from zero
    nn.backward({nn.embedding(ids_t, table_t, 1.7): dy_t})
    close(table_t.get_grad().np(), 2 * sums * scale, 2 * bound + 2 * U * np.abs(sums) * scale + 2 * U * bound, "twice")
    opt.zero_grad()
    nn.backward({nn.embedding(ids_t, table_t, 1.7): dy_t})
    assert_bit_exact(table_t.get_grad().np(), got, "again")


def test_embedding_many_tokens_and_shapes(nn_gpu):
    nn = nn_gpu
    rng = np.random.default_rng(5)
    ids = rng.integers(-1, 1000, (3, 50000)).astype(np.float32)
    table, dy = rng.standard_normal((1000, 4)).astype(np.float32), rng.standard_normal((3, 50000, 4)).astype(np.float32)
    table_t = nn.Tensor_from_value(table)
    trainable(nn, table_t)
    y = nn.embedding(nn.Tensor_from_value(ids), table_t)
    assert tuple(y.shape) == (3, 50000, 4)
    at = ids.astype(np.int64)
    assert_bit_exact(y.np(), np.where((at >= 0)[..., None], table[at], np.float32(0)))
    nn.backward({y: nn.Tensor_from_value(dy)})
    sums, size = np.zeros((1000, 4)), np.zeros((1000, 4))
    np.add.at(sums, at[at >= 0], dy[at >= 0].astype(np.float64))
    np.add.at(size, at[at >= 0], np.abs(dy[at >= 0]).astype(np.float64))
    close(table_t.get_grad().np(), sums, 200 * U * size, "gradient")         # (about 150 terms a row)


def test_embedding_in_a_table_of_more_than_2_32_values(nn_gpu):
    """Rows 2^32 values apart keep their own gradients, and are found again in the gradient."""
    nn = nn_gpu
    far, dim = 1 << 23, 516                                # (far * 512 = 2^32)
    ids = np.array([far + 1, 1, far, far + 1, 0, far * 512 // dim, far + 2], np.float32)
    dy = np.random.default_rng(11).standard_normal((7, dim)).astype(np.float32)
    table_t = nn.Tensor((far + 3, dim))
    trainable(nn, table_t)
    nn.backward({nn.embedding(nn.Tensor_from_value(ids), table_t): nn.Tensor_from_value(dy)})
    look = np.concatenate([ids, [far - 1, 2, far * 512 // dim + 1]]).astype(np.float32)
    got = nn.embedding(nn.Tensor_from_value(look), table_t.get_grad()).np()
    want = np.concatenate([dy, np.zeros((3, dim), np.float32)])
    want[0] = want[3] = dy[0] + dy[3]                      # (two terms: one rounding)
    assert_bit_exact(got, want)


@pytest.mark.parametrize("bad", [float("nan"), 7.0, 0.5, 3e9, float("inf")])
def test_bad_token_numbers_raise_at_the_next_read(nn_gpu, bad):
    nn = nn_gpu
    table_t = nn.Tensor_from_value(np.ones((7, 4), np.float32))
    trainable(nn, table_t)
    ids_t = nn.Tensor_from_value(np.array([1, bad, 6], np.float32))
    y = nn.embedding(ids_t, table_t)
    with pytest.raises(nn.LnnError, match="token number of an embedding"):
        y.np()
    assert_bit_exact(y.np()[:, 0], np.array([1, 0, 1], np.float32))          # the status is reported once
    nn.backward({y: nn.Tensor_from_value(np.ones((3, 4), np.float32))})
    with pytest.raises(nn.LnnError, match="gradient"):
        nn.devices.wait()
    assert_bit_exact(table_t.get_grad().np()[:, 0], np.array([0, 1, 0, 0, 0, 0, 1], np.float32))
    logits_t = nn.Tensor_from_value(np.zeros((3, 7), np.float32))
    with pytest.raises(nn.LnnError, match="row of logits"):
        nn.token_log_prob(logits_t, ids_t).np()
    if bad != 7.0:
        q = nn.Tensor_from_value(np.ones((3, 1, 6, 4), np.float32))
        with pytest.raises(nn.LnnError, match="length of a sequence"):
            nn.sink_attention(q, q, q, 4, lengths_t=ids_t).np()
        cache = nn.SinkCache(3, 1, 4, 1, 4)
        cache.set_lengths(ids_t)
        one = nn.Tensor_from_value(np.ones((3, 1, 4), np.float32))
        with pytest.raises(nn.LnnError, match="cached sequence"):
            nn.sink_attention_step(one, one, one, cache).np()
    nn.devices.wait()


# ---------------------------------------------------------------------------------------------
# probabilities of tokens
# ---------------------------------------------------------------------------------------------
def logit_bound(z, vocab):
    """How far log(sum exp(z - m)) may be off: the differences and their exponentials, chains of additions."""
    finite = np.where(np.isfinite(z), z, np.nan)
    span = np.nan_to_num(np.nanmax(finite, 1) - np.nanmin(np.where(finite > -1e30, finite, np.nan), 1))
    chain = vocab / 1024 + 16
    return U * (np.minimum(span, 100) + 8 * chain + 16)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 3), (5, 4), (7, 5), (37, 1003), (700, 257), (2, 8193), (3, 40001),
                                        (1, 200003), (600, 5000)])
def test_token_log_prob(nn_gpu, rows, vocab):
    nn = nn_gpu
    rng = np.random.default_rng(rows * vocab)
    z = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
    if vocab > 4:
        z[0, : vocab // 2] = -np.inf                      # tokens that are masked out
        z[-1, vocab // 2 + 1:] = np.finfo(np.float32).min
    ids = rng.integers(0, vocab, rows).astype(np.float32)
    ids[0], ids[-1] = vocab - 1, 0
    if rows > 4:
        ids[2] = -1
    dout = rng.standard_normal(rows).astype(np.float32)
    z_t, ids_t = nn.Tensor_from_value(z), nn.Tensor_from_value(ids)
    trainable(nn, z_t)
    y = nn.token_log_prob(z_t, ids_t)
    ref = torch.tensor(z, dtype=torch.float64, requires_grad=True)
    real = ids >= 0
    logp = torch.log_softmax(ref, 1)[torch.arange(rows), torch.tensor(ids).long().clamp(min=0)] * torch.tensor(real)
    logp.backward(torch.tensor(dout, dtype=torch.float64))
    want = logp.detach().numpy()
    off = logit_bound(z, vocab)
    close(y.np(), want, off + U * np.abs(want), "values")
    nn.backward({y: nn.Tensor_from_value(dout)})
    p = torch.softmax(ref.detach(), 1).numpy()
    # p with the error of its sum and of its own exponent, three products and a difference
    bound = np.abs(dout)[:, None] * (p * (off[:, None] + 8 * U) + 4 * U)
    close(z_t.get_grad().np(), ref.grad.numpy(), bound, "gradient")
    nn.backward({nn.token_log_prob(z_t, ids_t): nn.Tensor_from_value(dout)})
    close(z_t.get_grad().np(), 2 * ref.grad.numpy(), 2 * bound + 2 * U * np.abs(ref.grad.numpy()) + U * bound, "twice")


def test_token_log_prob_of_odd_rows(nn_gpu):
    nn = nn_gpu
    z = np.zeros((4, 9), np.float32)
    z[0, 4], z[1, 4], z[2] = np.nan, np.inf, -np.inf
    z_t = nn.Tensor_from_value(z.reshape(2, 2, 9))
    trainable(nn, z_t)
    y = nn.token_log_prob(z_t, nn.Tensor_from_value(np.array([[0, 1], [2, 3]], np.float32)))
    got = y.np()
    assert tuple(y.shape) == (2, 2) and np.isnan(got.reshape(-1)[:3]).all()
    close(got[1, 1], -math.log(9), 40 * U)
    y.backward()
    g = z_t.get_grad().np()
    assert np.isnan(g[0]).all() and np.isnan(g[1, 0]).all()
    close(g[1, 1], np.where(np.arange(9) == 3, 1.0, 0.0) - 1 / 9, 40 * U)


def test_logits_of_more_than_2_32_values(nn_gpu):
    nn = nn_gpu
    rows, vocab = 258, (1 << 24) - 1
    ids = np.arange(rows).astype(np.float32) * 50000
    z_t, ids_t = nn.Tensor((rows, vocab)), nn.Tensor_from_value(ids)
    z_t.fill(0.0)
    trainable(nn, z_t)
    y = nn.token_log_prob(z_t, ids_t)
    # a thread adds vocab / 8192 / 4 groups of ones, exactly; the rest is 16 roundings
    close(y.np(), np.full(rows, -math.log(vocab)), 40 * U)
    y.backward()
    # the gradient is 1 - 1 / vocab at the token and -1 / vocab elsewhere
    close(nn.token_log_prob(z_t.get_grad(), ids_t).np(), np.full(rows, 1 - math.log(vocab - 1 + math.e)), 60 * U)
    other = nn.Tensor_from_value((ids + 1).astype(np.float32))
    close(nn.token_log_prob(z_t.get_grad(), other).np(), np.full(rows, -math.log(vocab - 1 + math.e)), 60 * U)


@pytest.mark.parametrize("rows,vocab,kl,ref", [(1, 5, 0.0, False), (37, 1003, 0.05, True), (64, 300, 0.3, True), (9, 20000, 0.0, True),
                                               (350, 33, 1.0, True)])
def test_policy_loss(nn_gpu, rows, vocab, kl, ref):
    nn = nn_gpu
    rng = np.random.default_rng(rows + vocab)
    low, high = 0.1, 0.25
    z = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    ids = rng.integers(0, vocab, rows).astype(np.float32)
    if rows > 4:
        ids[3] = -2
    at = torch.tensor(ids).long().clamp(min=0)
    z64 = torch.tensor(z, dtype=torch.float64, requires_grad=True)
    logp = torch.log_softmax(z64, 1)[torch.arange(rows), at]
    # ratios on both sides of both borders, none within 1 % of one
    ratio = rng.choice([0.5, 0.8, 0.95, 1.0, 1.1, 1.2, 1.3, 2.0], rows)
    old = (logp.detach().numpy() - np.log(ratio)).astype(np.float32)
    refp = (logp.detach().numpy() + 0.5 * rng.standard_normal(rows)).astype(np.float32)
    adv, dout = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
    adv[0] = 0.0
    t = lambda x: torch.tensor(x, dtype=torch.float64)      # noqa: E731
    lo, hi = 1 - float(np.float32(low)), 1 + float(np.float32(high))
    r = torch.exp(logp - t(old))
    loss = -torch.minimum(r * t(adv), r.clamp(lo, hi) * t(adv))
    if kl:
        u = t(refp) - logp
        loss = loss + float(np.float32(kl)) * (torch.exp(u) - u - 1)
    loss = loss * t(ids >= 0)
    loss.backward(t(dout))
    z_t = nn.Tensor_from_value(z)
    trainable(nn, z_t)
    args = [nn.Tensor_from_value(x) for x in (ids, old, adv)]
    y = nn.policy_loss(z_t, *args, ref_t=nn.Tensor_from_value(refp) if ref else None, clip_low=low, clip_high=high, kl=kl)
    off = logit_bound(z, vocab)
    # d loss / d logp and its own derivative are at most |A| r + kl (1 + exp(u))
    steep = np.abs(adv) * ratio * 1.01 + kl * (1 + np.exp(np.abs(refp - logp.detach().numpy())))
    want = loss.detach().numpy()
    close(y.np(), want, steep * off + U * np.abs(want), "loss")
    nn.backward({y: nn.Tensor_from_value(dout)})
    p = torch.softmax(z64.detach(), 1).numpy()
    bound = (np.abs(dout) * steep)[:, None] * (p * (off[:, None] + 8 * U) + off[:, None] * np.abs((np.arange(vocab) == at.numpy()[:, None]) - p) + 4 * U * (p + (np.arange(vocab) == at.numpy()[:, None])))
    close(z_t.get_grad().np(), z64.grad.numpy(), bound, "gradient")
    if rows > 4:
        assert not z_t.get_grad().np()[3].any() and y.np()[3] == 0


def test_policy_loss_of_numbers_that_are_none(nn_gpu):
    """A row whose old logarithm, advantage or reference is NaN has a loss and a gradient of NaN; the others have not."""
    nn = nn_gpu
    z = np.random.default_rng(7).standard_normal((5, 33)).astype(np.float32)
    make = lambda *x: nn.Tensor_from_value(np.array(x, np.float32))      # noqa: E731
    nan = math.nan
    z_t = nn.Tensor_from_value(z)
    trainable(nn, z_t)
    y = nn.policy_loss(z_t, make(1, 2, 3, -1, 4), make(nan, -3, -3, nan, -3), make(0.5, nan, 0.5, nan, -0.5),
                       make(-3, -3, nan, nan, -3), kl=0.1)
    got = y.np()
    assert np.isnan(got[:3]).all() and got[3] == 0 and np.isfinite(got[4])
    y.backward()
    g = z_t.get_grad().np()
    assert np.isnan(g[:3]).all() and not g[3].any() and np.isfinite(g[4]).all() and g[4].any()
    # no probability before and no advantage: 0 times infinity
    assert np.isnan(nn.policy_loss(nn.Tensor_from_value(z[:1]), make(1), make(-math.inf), make(0)).np()).all()


def test_policy_loss_gradient_against_differences(nn_gpu):
    nn = nn_gpu
    rng = np.random.default_rng(8)
    z, way = rng.standard_normal((6, 50)).astype(np.float32), rng.standard_normal((6, 50)).astype(np.float32)
    ids = nn.Tensor_from_value(rng.integers(0, 50, 6).astype(np.float32))
    old, adv, ref = (nn.Tensor_from_value(x.astype(np.float32)) for x in (rng.uniform(-4.5, -3.5, 6), rng.standard_normal(6), rng.uniform(-4.5, -3.5, 6)))
    loss = lambda x: nn.policy_loss(x, ids, old, adv, ref, 1.0, 50.0, 0.2)       # noqa: E731  (nothing is clipped)
    z_t = nn.Tensor_from_value(z)
    trainable(nn, z_t)
    loss(z_t).backward()
    h = 2.0 ** -6
    up, down = (float(loss(nn.Tensor_from_value(z + s * h * way)).np().astype(np.float64).sum()) for s in (1, -1))
    slope = (z_t.get_grad().np().astype(np.float64) * way).sum()
    # third derivatives times h^2 / 6 (about 30 h^2), and 12 roundings of values below 50 over 2 h
    assert abs((up - down) / (2 * h) - slope) < 30 * h * h + 12 * 50 * U / h


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
def visible(T, S, window, sinks, lengths):
    p = np.arange(T)[:, None] + S - T
    j = np.arange(S)[None]
    m = (j <= p) & ((p - j < window) | (j < sinks))
    return torch.tensor(m[None] & (p[None] < np.asarray(lengths)[:, None, None]))[:, None]


def plain_attention(q, k, v, seen, scale):
    """64 bits; masked places may hold anything"""
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    x = (q @ k.transpose(-1, -2)) * scale
    any_ = seen.any(-1, keepdim=True)
    x = x.masked_fill(~seen, -math.inf).masked_fill(~any_, 0.0)
    return (torch.softmax(x, -1) * seen) @ v


def attention_bounds(q, k, v, do, seen, scale):
    """Element-wise bounds of o, dq, dk and dv.  A score is off by (D + 8) 2^-22 of the sum of its terms' magnitudes (fp32:
    D roundings of half a step; split operands: 3 * 2^-22 of it, and a few truncated accumulations), so a weight by
    twice that relative, and 2^-21 for its exponential; sums over n keys add n roundings."""
    g = q.shape[1] // k.shape[1]
    ka, va, qa, da = k.abs().repeat_interleave(g, 1), v.abs().repeat_interleave(g, 1), q.abs(), do.abs()
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    D, n = q.shape[-1], k.shape[2]
    s_off = (D + 8) * 2.0 ** -22 * scale * ((qa @ ka.transpose(-1, -2)) * seen).amax(-1, keepdim=True)
    any_ = seen.any(-1, keepdim=True)
    x = ((q @ kk.transpose(-1, -2)) * scale).masked_fill(~seen, -math.inf).masked_fill(~any_, 0.0)
    p = torch.softmax(x, -1) * seen
    w_off = 2 * s_off + 2.0 ** -20 + (n + 8) * 2.0 ** -23
    o_b = w_off * (p @ va)
    dp_mag = da @ va.transpose(-1, -2)                                     # bounds |dp| and, weighted, |delta|
    dp_mag = dp_mag + (p * dp_mag).sum(-1, keepdim=True)
    ds_b = p * dp_mag * (2 * w_off + (D + 8) * 2.0 ** -21) * scale
    ds_m = p * dp_mag * scale * (n * q.shape[1] + 8) * 2.0 ** -22          # the sums of the products behind
    fold = lambda t: t.reshape(t.shape[0], -1, g, *t.shape[2:]).sum(2)     # noqa: E731
    # dP - delta cancels where a row sees little else than one key: each is a sum of D products, off by D roundings of
    # their magnitudes, so that the gradients of q and k have this error beside one relative to themselves
    rest = p * dp_mag * scale * (D + 8) * U
    return (o_b, (ds_b + ds_m) @ ka, fold((ds_b + ds_m).transpose(-1, -2) @ qa),
            fold((p * (w_off + (n * q.shape[1] + 8) * 2.0 ** -22)).transpose(-1, -2) @ da),
            {"dq": float((rest @ ka).norm()), "dk": float(fold(rest.transpose(-1, -2) @ qa).norm())})


CASES = [
    # B, Hq, Hkv, T, S, D, window, sinks, lengths
    (1, 1, 1, 1, 1, 1, 1, 0, None),
    (1, 2, 1, 1, 5, 3, 2, 1, None),
    (2, 2, 2, 7, 7, 16, 3, 0, (7, 0)),
    (1, 4, 2, 63, 63, 32, 100, 0, None),
    (1, 2, 2, 64, 64, 64, 64, 4, None),
    (3, 3, 1, 65, 65, 40, 16, 2, (65, 64, 1)),
    (2, 6, 3, 130, 130, 80, 33, 5, (130, 77)),
    (1, 2, 1, 100, 300, 128, 50, 3, None),
    (2, 2, 2, 200, 333, 64, 90, 70, (333, 140)),
    (1, 1, 1, 257, 257, 96, 1, 0, None),
    (1, 2, 1, 257, 257, 128, 1, 1, None),
    (1, 3, 3, 70, 70, 200, 20, 2, None),
    (2, 2, 1, 40, 90, 256, 1000, 500, (90, 60)),
    (1, 2, 2, 520, 520, 64, 130, 130, None),
    (1, 1, 1, 700, 700, 17, 64, 3, (640,)),
    (2, 4, 2, 384, 384, 128, 128, 4, (384, 383)),
    # more tiles of 128 rows than the device has SMs
    (3, 16, 8, 500, 530, 24, 90, 2, (530, 77, 400)),
    (2, 24, 12, 900, 900, 66, 300, 6, None),
    # few tiles that see many keys: cut over several works, the parts merged
    (1, 1, 1, 1500, 1500, 64, 1500, 0, None),
    (2, 1, 1, 700, 1100, 96, 2000, 0, (1100, 650)),
    (1, 2, 1, 129, 4000, 128, 3900, 130, None),
    (1, 4, 4, 1, 5000, 64, 4000, 3, None),
    # a sequence of which no query is real
    (2, 2, 2, 50, 200, 64, 30, 2, (150, 200)),
    # more heads than the tensor-core kernels have counters for
    (2100, 4, 2, 66, 66, 4, 20, 1, None),
]


def attention_inputs(case, seed=0):
    B, Hq, Hkv, T, S, D, window, sinks, lengths = case
    rng = np.random.default_rng(seed + T * S + D)
    make = lambda *s: rng.standard_normal(s).astype(np.float32)      # noqa: E731
    return (make(B, Hq, T, D), make(B, Hkv, S, D), make(B, Hkv, S, D), make(B, Hq, T, D)), lengths or (S,) * B


@pytest.mark.parametrize("case", CASES)
def test_sink_attention(nn_gpu, case):
    nn = nn_gpu
    B, Hq, Hkv, T, S, D, window, sinks, lengths = case
    (q, k, v, do), lens = attention_inputs(case)
    seen, scale = visible(T, S, window, sinks, lens), D ** -0.5
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = plain_attention(*r, seen, scale)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = attention_bounds(*[x.detach() for x in r], d64, seen, scale)
    # padded keys and rows may hold anything, and so may keys that no query sees
    for b, n in enumerate(lens):
        k[b, :, n:] = np.nan
        v[b, :, n:] = np.inf
        p = np.arange(T) + S - T
        q[b, :, p >= n] = np.nan
        do[b, :, p >= n] = np.inf
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *t)
    lens_t = nn.Tensor_from_value(np.array(lens, np.float32)) if lengths else None
    y = nn.sink_attention(*t, window, sinks, lengths_t=lens_t)
    do_t = nn.Tensor_from_value(do)
    nn.backward({y: do_t})
    got = [y.np()] + [x.get_grad().np() for x in t]
    for name, g, w, b in zip(("o", "dq", "dk", "dv"), got, [o.detach()] + [x.grad for x in r], bounds):
        close(g, w.numpy(), b.detach().numpy() + 1e-30, name)
        norm = float(w.norm())
        assert np.linalg.norm(g - w.numpy()) <= 1e-5 * norm + bounds[4].get(name, 0.0) + 1e-30, (name, np.linalg.norm(g - w.numpy()), norm)
    # a second pass adds to the gradients, one value at a time: a rounding of each sum
    nn.backward({nn.sink_attention(*t, window, sinks, lengths_t=lens_t): do_t})
    for name, g, x in zip(("dq", "dk", "dv"), got[1:], t):
        assert_bit_exact(x.get_grad().np(), g + g, name)


@pytest.mark.parametrize("D", [64, 72])
@pytest.mark.parametrize("what", ["empty", "outlier"])
def test_works_of_other_kernels_between_long_ones(nn_gpu, D, what):
    """Six tiles of 128 heads, for which a block has two between two full ones that see nothing, or that are of heads with a
    value that their split form does not hold (in a row that the guess of the scale does not look at)."""
    nn = nn_gpu
    B, H, S, window, sinks = 8, 16, 768, 100, 3
    rng = np.random.default_rng(31)
    q, k, v, do = (rng.standard_normal((B, H, S, D)).astype(np.float32) for _ in range(4))
    if what == "empty":
        lens, full = [768, 0, 0, 768, 0, 0, 0, 300], [0, 3, 7]
    else:
        lens, full = [768] * 7 + [300], [0, 2, 3, 7]
        k[[1, 2, 4, 5, 6], :, 5, 3] = 2000.0
    seen, scale = visible(S, S, window, sinks, [lens[b] for b in full]), D ** -0.5
    r = [torch.tensor(x[full], dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = plain_attention(*r, seen, scale)
    d64 = torch.tensor(do[full], dtype=torch.float64)
    o.backward(d64)
    bounds = attention_bounds(*[x.detach() for x in r], d64, seen, scale)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *t)
    y = nn.sink_attention(*t, window, sinks, lengths_t=nn.Tensor_from_value(np.array(lens, np.float32)))
    nn.backward({y: nn.Tensor_from_value(do)})
    rest = [b for b in range(B) if lens[b] == 0]
    for name, g, w, b in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach()] + [x.grad for x in r], bounds):
        g = g.np()
        assert not g[rest].any(), name
        close(g[full], w.numpy(), b.detach().numpy() + 1e-30, name)


def test_sink_attention_masked_places_hold_anything(nn_gpu):
    """Keys that a row does not see do not reach it, whatever they hold, even where its neighbours see them."""
    nn = nn_gpu
    q, k, v = (np.random.default_rng(3).standard_normal((1, 2, 300, 64)).astype(np.float32) for _ in range(3))
    clean = nn.sink_attention(*[nn.Tensor_from_value(x) for x in (q, k, v)], 20).np()
    for where, value in ((100, np.nan), (100, np.inf), (131, -np.inf)):
        k2, v2 = k.copy(), v.copy()
        k2[:, :, where] = value
        v2[:, :, where] = value
        t = [nn.Tensor_from_value(x) for x in (q, k2, v2)]
        trainable(nn, *t)
        y = nn.sink_attention(*t, 20)
        got = y.np()
        away = np.r_[0:where, where + 20:300]
        close(got[:, :, away], clean[:, :, away], 1e-5, "rows that do not see it")
        do = np.ones((1, 2, 300, 64), np.float32)
        do[:, :, where:where + 20] = 0
        nn.backward({y: nn.Tensor_from_value(do)})
        assert np.isfinite(t[0].get_grad().np()[:, :, away]).all()
        far = np.r_[0:where - 20, where + 40:300]
        assert np.isfinite(t[1].get_grad().np()[:, :, far]).all() and np.isfinite(t[2].get_grad().np()[:, :, far]).all()


@pytest.mark.parametrize("scale_q,scale_v", [(1e-18, 1e18), (1e4, 1e-20), (0.0, 1.0)])
def test_sink_attention_magnitudes(nn_gpu, scale_q, scale_v):
    nn = nn_gpu
    (q, k, v, do), lens = attention_inputs((1, 2, 1, 150, 150, 64, 60, 4, None))
    q, v, do = q * np.float32(scale_q), v * np.float32(scale_v), do * np.float32(1e-6)
    k = k * np.float32(1e-3)
    seen = visible(150, 150, 60, 4, lens)
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = plain_attention(*r, seen, 0.3)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = attention_bounds(*[x.detach() for x in r], d64, seen, 0.3)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *t)
    y = nn.sink_attention(*t, 60, 4, scale=0.3)
    nn.backward({y: nn.Tensor_from_value(do)})
    for name, g, w, b in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach()] + [x.grad for x in r], bounds):
        close(g.np(), w.numpy(), b.detach().numpy() + 1e-37, name)


def test_sink_attention_one_tensor_in_three_places(nn_gpu):
    nn = nn_gpu
    x = np.random.default_rng(4).standard_normal((2, 2, 90, 32)).astype(np.float32)
    do = np.random.default_rng(5).standard_normal(x.shape).astype(np.float32)
    r = torch.tensor(x, dtype=torch.float64, requires_grad=True)
    seen = visible(90, 90, 40, 2, (90, 90))
    plain_attention(r, r, r, seen, 32 ** -0.5).backward(torch.tensor(do, dtype=torch.float64))
    t = nn.Tensor_from_value(x.reshape(4, 90, 32))
    trainable(nn, t)
    a = t.reshape(x.shape)
    y = nn.sink_attention(a, a, t.reshape(x.shape), 40, 2)
    nn.backward({y: nn.Tensor_from_value(do)})
    assert np.linalg.norm(t.get_grad().np().reshape(x.shape) - r.grad.numpy()) <= 1e-5 * float(r.grad.norm())


@pytest.mark.parametrize("D", [1, 64, 128])
def test_sink_attention_with_rows_of_nothing(nn_gpu, D):
    """Rows of zeros, and some of tiny values, in each of the inputs."""
    nn = nn_gpu
    case = (1, 4, 2, 300, 300, D, 150, 4, None)
    inputs, lens = attention_inputs(case)
    for i, x in enumerate(inputs):
        x[:, :, i::7] = 0.0
        x[:, :, i + 3::11] *= np.float32(1e-6)
    q, k, v, do = inputs
    seen, scale = visible(300, 300, 150, 4, lens), D ** -0.5
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (q, k, v)]
    o = plain_attention(*r, seen, scale)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = attention_bounds(*[x.detach() for x in r], d64, seen, scale)
    # Beside errors relative to the terms: lo ends at fp16's smallest step, 2^-24, where the head's largest value is 2^8 or more, so
    # that an operand is off by step = 2^-33 of its largest.  A weight is off by `weight` through q and k then, dP - delta by D
    # products of which each has two such operands, and what they are multiplied with (k: 1 weight in all, q and dO: n) by one.
    step, n = 2.0 ** -33, 300 * 2
    Q, K, V, DO = (float(np.abs(x).max()) for x in inputs)
    weight = 2 * (2 * step * scale * D * Q * K)
    ds = scale * D * DO * V * (2 * weight + 2 * step + 2 * step)
    rest = (V * (weight + step), K * ds, n * Q * ds, n * DO * (weight + step))
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *t)
    y = nn.sink_attention(*t, 150, 4)
    nn.backward({y: nn.Tensor_from_value(do)})
    for name, g, w, b, c in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach()] + [x.grad for x in r], bounds,
                                rest):
        close(g.np(), w.numpy(), b.detach().numpy() + c, name)


def test_sink_attention_with_a_negative_scale(nn_gpu):
    nn = nn_gpu
    (q, k, v, do), lens = attention_inputs((1, 2, 1, 150, 150, 64, 60, 4, None))
    seen = visible(150, 150, 60, 4, lens)
    r = [torch.tensor(x, dtype=torch.float64, requires_grad=True) for x in (-q, k, v)]
    o = plain_attention(*r, seen, 0.3)
    d64 = torch.tensor(do, dtype=torch.float64)
    o.backward(d64)
    bounds = attention_bounds(*[x.detach() for x in r], d64, seen, 0.3)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *t)
    y = nn.sink_attention(*t, 60, 4, scale=-0.3)
    nn.backward({y: nn.Tensor_from_value(do)})
    for name, g, w, b in zip(("o", "dq", "dk", "dv"), [y] + [x.get_grad() for x in t], [o.detach(), -r[0].grad, r[1].grad, r[2].grad],
                             bounds):
        close(g.np(), w.numpy(), b.detach().numpy() + 1e-30, name)


@pytest.mark.parametrize("bad", [float("nan"), 0.5, 2000.0])
def test_bad_lengths_of_long_sequences(nn_gpu, bad):
    """Kernels in tiles end early; the next call is right again."""
    nn = nn_gpu
    case = (2, 2, 1, 300, 300, 64, 120, 4, None)
    (q, k, v, do), _ = attention_inputs(case)
    t = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *t)
    do_t = nn.Tensor_from_value(do)
    want = nn.sink_attention(*t, 120, 4)
    nn.backward({want: do_t})
    want, grads = want.np(), [x.get_grad().np() for x in t]
    for x in t:
        x.zero_grad()
    y = nn.sink_attention(*t, 120, 4, lengths_t=nn.Tensor_from_value(np.array([300, bad], np.float32)))
    nn.backward({y: do_t})
    with pytest.raises(nn.LnnError, match="length of a sequence"):
        y.np()
    for x in t:
        x.zero_grad()
    y = nn.sink_attention(*t, 120, 4)
    nn.backward({y: do_t})
    assert_bit_exact(y.np(), want)
    for x, g in zip(t, grads):
        assert_bit_exact(x.get_grad().np(), g)


def test_sink_attention_only_some_gradients(nn_gpu):
    nn = nn_gpu
    (q, k, v, do), _ = attention_inputs((1, 2, 1, 70, 70, 64, 30, 4, None))
    full = [nn.Tensor_from_value(x) for x in (q, k, v)]
    trainable(nn, *full)
    nn.backward({nn.sink_attention(*full, 30, 4): nn.Tensor_from_value(do)})
    for which in range(3):
        t = [nn.Tensor_from_value(x) for x in (q, k, v)]
        trainable(nn, t[which])
        nn.backward({nn.sink_attention(*t, 30, 4): nn.Tensor_from_value(do)})
        for i in range(3):
            assert t[i].has_grad() == (i == which)
        assert_bit_exact(t[which].get_grad().np(), full[which].get_grad().np())


def test_sink_attention_gradient_against_differences(nn_gpu):
    nn = nn_gpu
    rng = np.random.default_rng(6)
    x = [rng.standard_normal((1, 2, 33, 8)).astype(np.float32) for _ in range(3)]
    way = [rng.standard_normal((1, 2, 33, 8)).astype(np.float32) for _ in range(3)]
    f = lambda *t: nn.sink_attention(*t, 9, 2)      # noqa: E731
    t = [nn.Tensor_from_value(a) for a in x]
    trainable(nn, *t)
    f(*t).backward()
    slope = sum((a.get_grad().np().astype(np.float64) * w).sum() for a, w in zip(t, way))
    h = 2.0 ** -7
    up, down = (f(*[nn.Tensor_from_value(a + s * h * w) for a, w in zip(x, way)]).np().astype(np.float64).sum() for s in (1, -1))
    # 528 values below 4, each off by 2^-20 of it (random signs: sqrt(528) of them), and h^2 / 6 of their third derivatives
    assert abs((up - down) / (2 * h) - slope) < 23 * 4 * 2.0 ** -20 / h + 528 * h * h


# ---------------------------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,Hq,Hkv,D,window,sinks", [
    (1, 1, 1, 1, 1, 0), (2, 2, 1, 3, 5, 2), (3, 6, 3, 64, 20, 4), (2, 8, 1, 80, 7, 0), (1, 5, 1, 128, 40, 3), (2, 3, 3, 130, 9, 1),
    (1, 4, 2, 256, 33, 5), (1, 16, 2, 96, 12, 1), (2, 2, 2, 32, 700, 30), (2, 2, 2, 96, 20, 3)])
def test_steps_equal_attention_over_the_whole(nn_gpu, B, Hq, Hkv, D, window, sinks):
    """A prompt into the cache, then one token after another, past the end of the ring."""
    nn = nn_gpu
    total = min(2 * window + sinks + 9, 760)
    prompt = total - min(total - 1, 40)
    rng = np.random.default_rng(D + window)
    q, k, v = (rng.standard_normal((B, h, total, D)).astype(np.float32) for h in (Hq, Hkv, Hkv))
    lens = [max(1, prompt - 3 * b) for b in range(B)]
    cache = nn.SinkCache(B, Hkv, window, sinks, D)
    for t in (cache.k, cache.v):
        t.fill(float("nan"))                               # slots that are not in use may hold anything
    kp, vp = k[:, :, :prompt].copy(), v[:, :, :prompt].copy()
    cache.store(nn.Tensor_from_value(kp), nn.Tensor_from_value(vp), nn.Tensor_from_value(np.array(lens, np.float32)))
    assert cache.lengths.np().tolist() == lens
    r = [torch.tensor(x, dtype=torch.float64) for x in (q, k, v)]
    want = plain_attention(*r, visible(total, total, window, sinks, (total,) * B), D ** -0.5).numpy()
    size = float(np.abs(v).max())
    # scores off by (D + 8) 2^-23 of their terms' magnitudes at most, twice that and 2^-20 for a weight; n keys
    bound = size * (2 * (D + 8) * 2.0 ** -23 * D ** -0.5 * float((np.abs(q).sum(-1).max() * np.abs(k).max())) + 2.0 ** -20 + (window + sinks) * U)
    for step in range(total - max(lens)):
        at = [n + step for n in lens]
        pick = lambda x: nn.Tensor_from_value(np.stack([x[b, :, at[b]] for b in range(B)]))      # noqa: E731
        y = nn.sink_attention_step(pick(q), pick(k), pick(v), cache)
        close(y.np(), np.stack([want[b, :, at[b]] for b in range(B)]), bound, f"step {step}")
    assert cache.lengths.np().tolist() == [n + 1 for n in at]


def test_step_over_a_long_cache(nn_gpu):
    """The slots of one head cut over the blocks of a cluster, with a share that is empty."""
    nn = nn_gpu
    rng = np.random.default_rng(9)
    for length in (0, 1, 31, 700, 1023, 1029, 5000):
        window, sinks, D = 1020, 9, 64
        k, v = (rng.standard_normal((1, 1, window + sinks, D)).astype(np.float32) for _ in range(2))
        q1, k1, v1 = (rng.standard_normal((1, h, D)).astype(np.float32) for h in (2, 1, 1))
        cache = nn.SinkCache(1, 1, window, sinks, D)
        cache.k.set(k)
        cache.v.set(v)
        cache.set_lengths(length)
        y = nn.sink_attention_step(*[nn.Tensor_from_value(x) for x in (q1, k1, v1)], cache)
        slot = length if length < sinks else sinks + (length - sinks) % window
        k[:, :, slot], v[:, :, slot] = k1, v1
        assert_bit_exact(cache.k.np(), k)
        assert_bit_exact(cache.v.np(), v)
        n = min(length + 1, window + sinks)
        r = [torch.tensor(x, dtype=torch.float64) for x in (q1[:, :, None], k[:, :, :n], v[:, :, :n])]
        want = plain_attention(*r, torch.ones(1, 1, 1, n, dtype=torch.bool), D ** -0.5).numpy()[:, :, 0]
        close(y.np(), want, 5 * (72 * 2.0 ** -22 * 10 + 2.0 ** -20 + n * U), f"length {length}")


def test_step_over_a_cache_of_more_than_2_32_values(nn_gpu):
    """All old keys and values are zero: n of them and the new ones share the weights 1 : exp(s)."""
    nn = nn_gpu
    slots, D = 1 << 24, 160
    cache = nn.SinkCache(2, 1, slots - 5, 5, D)
    cache.k.fill(0.0)
    cache.v.fill(0.0)
    lengths = np.array([10, slots - 3])
    cache.set_lengths(lengths)
    one = np.ones((2, 1, D), np.float32)
    score = np.log([10, 2.0 ** 24]).astype(np.float32)             # half of the weight for the first new key
    key = one * (score[:, None, None] / D)
    value = np.random.default_rng(12).standard_normal((2, 2, 1, D)).astype(np.float32)
    for step in range(2):
        y = nn.sink_attention_step(*[nn.Tensor_from_value(x) for x in (one, key, value[step])], cache, scale=1.0).np()
        w = np.exp(np.float64(D) * key[:, :, :1])
        want = value[:step + 1].astype(np.float64).sum(0) * w / (lengths[:, None, None] + w * (step + 1))
        # the score is off by D + 8 roundings, the weight by that, a sum of whole numbers up to 2^24 by 16 roundings
        close(y, want, np.abs(value).max() * 2 * ((D + 8) * U * 17 + 16 * U), f"step {step}")
    assert cache.lengths.np().tolist() == (lengths + 2).tolist()


def test_places_that_are_not_in_use_stay_as_they_are(nn_gpu):
    nn = nn_gpu
    rng = np.random.default_rng(10)
    cache = nn.SinkCache(3, 2, 4, 1, 8)
    k, v = (rng.standard_normal((3, 2, 6, 8)).astype(np.float32) for _ in range(2))
    cache.k.fill(3.0)
    cache.v.fill(4.0)
    cache.set_lengths([7, 2, -1])
    cache.store(nn.Tensor_from_value(k), nn.Tensor_from_value(v), nn.Tensor_from_value(np.array([3, -1, 6], np.float32)))
    assert cache.lengths.np().tolist() == [3, 2, 6]
    got = cache.k.np()
    assert_bit_exact(got[0, :, :3], k[0, :, :3])
    assert (got[0, :, 3:] == 3).all() and (got[1] == 3).all()
    assert_bit_exact(got[2], k[2][:, [0, 5, 2, 3, 4]])       # positions 1 and 5 share a slot
    cache.set_lengths([3, -1, 6])
    one = nn.Tensor_from_value(np.ones((3, 2, 8), np.float32))
    y = nn.sink_attention_step(one, one, one, cache).np()
    assert (y[1] == 0).all() and (y[0] != 0).any() and (cache.k.np()[1] == 3).all() and (cache.v.np()[1] == 4).all()
    assert cache.lengths.np().tolist() == [4, -1, 7]
    cache.set_lengths(-1)
    assert not nn.sink_attention_step(one, one, one, cache).np().any()


# ---------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------
def test_a_small_model_from_tokens_to_the_loss(nn_gpu):
    """Embedding, projections, attention, logits, policy loss: loss and all gradients of one training step; then the same
    model answers from a prompt, token by token, with the logits of the whole."""
    nn = nn_gpu
    V, E, H, D, B, T, window, sinks = 50, 24, 2, 16, 2, 21, 6, 2
    rng = np.random.default_rng(11)
    np.random.seed(12)

    class Small(nn.Module):
        def __init__(self):
            self.emb = nn.Embedding(V, E, scale=2.0, weight_initializer=nn.initializer.RandomNormal(0.0, 0.5))
            self.q, self.k, self.v, self.o = (nn.Dense(i, o, use_bias=False) for i, o in
                                              ((E, 2 * H * D), (E, H * D), (E, H * D), (2 * H * D, V)))

    net = Small()
    emb, layers = net.emb, {n: getattr(net, n) for n in "qkvo"}
    params = [emb.weight] + [layers[n].weight for n in "qkvo"]
    opt = nn.optimizer.SGD(net.trainables())
    ids = rng.integers(0, V, (B, T)).astype(np.float32)
    lens = np.array([T, T - 5], np.float32)
    ids[1, T - 5:] = -1
    target = np.where(ids < 0, -1, rng.integers(0, V, (B, T))).astype(np.float32)
    old, adv, ref = rng.uniform(-6, -3, (B, T)).astype(np.float32), rng.standard_normal((B, T)).astype(np.float32), rng.uniform(-6, -3, (B, T)).astype(np.float32)

    def heads(x, h, t):
        return x.reshape((B, t, h, D)).transpose((0, 2, 1, 3))

    def qkv(x):
        t = x.shape[1]
        flat = x.reshape((B * t, E))
        return [heads(layers[n](flat), h, t) for n, h in (("q", 2 * H), ("k", H), ("v", H))]

    def model(ids_t, lens_t):
        q, k, v = qkv(emb(ids_t))
        o = nn.sink_attention(q, k, v, window, sinks, lengths_t=lens_t)
        return layers["o"](o.transpose((0, 2, 1, 3)).reshape((B * T, 2 * H * D))), k, v

    t = nn.Tensor_from_value
    logits, _, _ = model(t(ids), t(lens))
    loss = nn.policy_loss(logits, t(target), t(old), t(adv), t(ref), 0.2, 0.2, 0.1).sum()
    loss.backward()

    w = [torch.tensor(p.np(), dtype=torch.float64, requires_grad=True) for p in params]
    at = torch.tensor(ids).long()
    x = torch.where(at[..., None] >= 0, w[0][at.clamp(min=0)] * 2.0, 0.0)
    split = lambda m, h: (x @ m).reshape(B, T, h, D).transpose(1, 2)      # noqa: E731
    o = plain_attention(split(w[1], 2 * H), split(w[2], H), split(w[3], H), visible(T, T, window, sinks, lens.astype(int)), D ** -0.5)
    z = (o.transpose(1, 2).reshape(B * T, 2 * H * D) @ w[4])
    tt = torch.tensor(target.reshape(-1)).long()
    logp = torch.log_softmax(z, 1)[torch.arange(B * T), tt.clamp(min=0)]
    f = lambda a: torch.tensor(a.reshape(-1), dtype=torch.float64)        # noqa: E731
    r, u = torch.exp(logp - f(old)), f(ref) - logp
    each = -torch.minimum(r * f(adv), r.clamp(0.8, 1.2) * f(adv)) + 0.1 * (torch.exp(u) - u - 1)
    total = (each * (tt >= 0)).sum()
    total.backward()
    close(loss.np()[0], float(total.detach()), 1e-4 * float(each.detach().abs().sum()), "loss")
    for p, a in zip(params, w):
        g = p.get_grad().np()
        assert np.linalg.norm(g - a.grad.numpy()) <= 1e-4 * float(a.grad.norm()), np.linalg.norm(g - a.grad.numpy()) / float(a.grad.norm())

    with nn.optimizer.freeze():
        whole, _, _ = model(t(np.where(ids < 0, 0, ids)), t(np.full(B, T, np.float32)))
        whole = whole.np().reshape(B, T, V)
        first = T - 8
        cache = nn.SinkCache(B, H, window, sinks, D)
        filled = np.where(ids < 0, 0, ids)
        _, k, v = qkv(emb(t(filled[:, :first])))
        cache.store(k, v)
        for p in range(first, T):
            q, k, v = [a.reshape((B, -1, D)) for a in qkv(emb(t(filled[:, p:p + 1])))]
            o = nn.sink_attention_step(q, k, v, cache)
            got = layers["o"](o.reshape((B, 2 * H * D))).np()
            close(got, whole[:, p], 1e-5 * np.abs(whole).max(), f"position {p}")
    opt.zero_grad()
