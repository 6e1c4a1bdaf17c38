"""CPU: the operators on tokens and sequences on the host: refusals, the tape, and what is asked of the library."""
import numpy as np
import pytest

import litenn_b200 as nn
from fake_device import fake_device
from litenn_b200 import _lib


@pytest.fixture
def fake():
    with fake_device() as f:
        yield f


def T(*shape):
    return nn.Tensor(shape)


def refused(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def test_refusals_of_embedding(fake):
    refused("table_t must be", nn.embedding, T(3), T(4, 5, 6))
    refused("must be a Tensor", nn.embedding, np.zeros(3, np.float32), T(4, 5))
    refused("must be a Tensor", nn.embedding, T(3), None)
    refused("exact in fp32", nn.embedding, T(3), T((1 << 24) + 1, 1))
    assert "lnn_embedding_fwd" not in fake.calls
    assert tuple(nn.embedding(T(2, 3), T(4, 5)).shape) == (2, 3, 5)


def test_refusals_of_the_losses(fake):
    z, n = T(2, 3, 7), T(2, 3)
    refused("rank 2", nn.token_log_prob, T(7), T(1))
    refused("6 elements", nn.token_log_prob, z, T(7))
    refused("must be a Tensor", nn.token_log_prob, z, [1, 2])
    refused("old_t must have", nn.policy_loss, z, n, T(2), n)
    refused("advantage_t must have", nn.policy_loss, z, n, n, T(7))
    refused("ref_t must have", nn.policy_loss, z, n, n, n, T(1), kl=0.1)
    refused("old_t must be a Tensor", nn.policy_loss, z, n, None, n)
    refused("needs ref_t", nn.policy_loss, z, n, n, n, kl=0.1)
    refused("negative", nn.policy_loss, z, n, n, n, n, kl=-0.1)
    refused("negative", nn.policy_loss, z, n, n, n, n, kl=float("nan"))
    for low, high in ((-0.1, 0.2), (1.1, 0.2), (0.2, -0.2), (float("nan"), 0.2), (0.2, float("inf"))):
        refused("cannot be clipped", nn.policy_loss, z, n, n, n, clip_low=low, clip_high=high)
    assert not any(c.startswith("lnn_token") or c.startswith("lnn_policy") for c in fake.calls)
    assert tuple(nn.policy_loss(z, n, n, n).shape) == (2, 3) and tuple(nn.token_log_prob(T(1, 7), T(1)).shape) == (1,)


def test_refusals_of_attention(fake):
    q, k = T(2, 4, 5, 8), T(2, 2, 9, 8)
    f = nn.sink_attention
    refused("expected q", f, T(4, 5, 8), k, k, 3)
    refused("expected q", f, q, k, T(2, 2, 9, 4), 3)
    refused("does not go with", f, T(3, 4, 5, 8), k, k, 3)
    refused("does not go with", f, T(2, 3, 5, 8), k, k, 3)
    refused("does not go with", f, T(2, 4, 5, 4), k, k, 3)
    refused("5 queries over 4 keys", f, q, T(2, 2, 4, 8), T(2, 2, 4, 8), 3)
    refused("window", f, q, k, k, 0)
    refused("window", f, q, k, k, 2.5)
    refused("sinks", f, q, k, k, 3, -1)
    refused("must be finite", f, q, k, k, 3, scale=float("inf"))
    refused("at most 256", f, T(1, 1, 1, 257), T(1, 1, 1, 257), T(1, 1, 1, 257), 3)
    refused("2 elements", f, q, k, k, 3, lengths_t=T(3))
    refused("must be a Tensor", f, q, k, k, 3, lengths_t=[9, 9])
    assert "lnn_sink_attn_fwd" not in fake.calls


def test_refusals_of_the_cache(fake):
    for bad in ((0, 1, 1, 0, 1), (1, 0, 1, 0, 1), (1, 1, 0, 0, 1), (1, 1, 1, -1, 1), (1, 1, 1, 0, 257), (1, 1, 1 << 24, 1, 1)):
        with pytest.raises(ValueError):
            nn.SinkCache(*bad)
    c = nn.SinkCache(2, 3, 4, 1, 8)
    kv = T(2, 3, 8)
    refused("expected k and v", nn.sink_attention_step, T(2, 3, 8), T(2, 3, 4), kv, c)
    refused("does not go with", nn.sink_attention_step, T(2, 4, 8), kv, kv, c)
    refused("does not go with", nn.sink_attention_step, T(1, 3, 8), kv, kv, c)
    refused("must be finite", nn.sink_attention_step, T(2, 3, 8), kv, kv, c, scale=float("nan"))
    refused("SinkCache", nn.sink_attention_step, T(2, 3, 8), kv, kv, None)
    refused("expected k and v", c.store, T(2, 3, 4), T(2, 3, 4))
    refused("2 elements", c.store, T(2, 3, 4, 8), T(2, 3, 4, 8), T(3))
    refused("from itself", c.store, c.k, T(2, 3, 5, 8))
    refused("from itself", c.store, T(2, 3, 5, 8), T(2, 3, 5, 8), c.lengths)
    one = nn.SinkCache(2, 3, 1, 0, 8)
    refused("own memory", nn.sink_attention_step, T(2, 3, 8), one.k.reshape((2, 3, 8)), kv, one)
    refused("elements", c.set_lengths, [1, 2, 3])
    assert not any("step" in x or "store" in x for x in fake.calls)


def test_lengths_change_places_only_after_a_step_that_ran(fake):
    c = nn.SinkCache(2, 1, 4, 1, 8)
    c.set_lengths([3, 5])
    kv = T(2, 1, 8)
    before = c.lengths
    fake.fail["lnn_sink_attn_step"] = _lib.E_CUDA
    with pytest.raises(_lib.LnnError):
        nn.sink_attention_step(kv, kv, kv, c)
    assert c.lengths is before and before.np().tolist() == [3, 5]
    nn.sink_attention_step(kv, kv, kv, c)
    assert c.lengths is not before
    with nn.devices._shallow_mode():
        now = c.lengths
        assert tuple(nn.sink_attention_step(kv, kv, kv, c).shape) == (2, 1, 8)
        assert c.lengths is now


def test_the_gradients_of_attention_are_asked_for_together(fake):
    q, k, v = T(1, 2, 3, 4), T(1, 2, 3, 4), T(1, 2, 3, 4)
    nn.optimizer.SGD([q, k, v])
    fake.calls.clear()
    nn.sink_attention(q, k, v, 2).backward()
    assert fake.calls.count("lnn_sink_attn_bwd") == 1 and all(t.has_grad() for t in (q, k, v))
    # a view of one tensor in all three places: two gradients go to memory of their own and are added
    x = T(2, 3, 4)
    nn.optimizer.SGD([x])
    a = x.reshape((1, 2, 3, 4))
    fake.calls.clear()
    nn.sink_attention(a, a, x.reshape((1, 2, 3, 4)), 2).backward()
    assert fake.calls.count("lnn_sink_attn_bwd") == 1 and fake.calls.count("lnn_binary_fwd") == 2
    # only the keys are trained
    k = T(1, 2, 3, 4)
    nn.optimizer.SGD([k])
    q = T(1, 2, 3, 4)
    nn.sink_attention(q, k, q, 2).backward()
    assert k.has_grad() and not q.has_grad()


def test_other_grad_functions_of_an_attention_result_run_too(fake):
    q, other = T(1, 2, 3, 4), T(1,)
    nn.optimizer.SGD([q, other])
    y = nn.sink_attention(q, q, q, 2)
    seen = []
    y._assign_gradfn(q, lambda O_t, dO_t: seen.append("q"))
    y._assign_gradfn(other, lambda O_t, dO_t: seen.append("other"))
    y.backward()
    assert sorted(seen) == ["other", "q"]


def test_an_embedding_module_saves_its_table(fake):
    m = nn.Embedding(5, 3, scale=2.0, weight_initializer=nn.initializer.Scalar(1.0))
    assert [t.get_name() for t in m.trainables()] == ["Embedding.weight"]
    assert tuple(m(T(2, 2)).shape) == (2, 2, 3)
    assert "num_tokens:5" in str(m)


@pytest.mark.parametrize("number", [3, 3.0, np.int64(3), np.float32(3), np.array(3)])
def test_one_number_is_the_length_of_all(fake, number):
    c = nn.SinkCache(2, 1, 4, 1, 8)
    c.set_lengths(number)
    assert c.lengths.np().tolist() == [3, 3]


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), -float("inf")])
def test_spans_that_are_not_finite_are_refused(fake, bad):
    q = T(1, 1, 3, 4)
    refused("window", nn.sink_attention, q, q, q, bad)
    refused("sinks", nn.sink_attention, q, q, q, 2, bad)
    refused("window", nn.SinkCache, 1, 1, bad, 0, 4)
