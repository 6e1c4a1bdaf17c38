"""Operators on tokens and sequences: rows of a table, attention with a sliding window and a few first tokens that stay
visible, its cache for one token after another, the logarithm of a token's probability and the clipped policy loss.

They follow the op layer (ops.py): shapes are checked on the host, a result tensor with its grad functions is made, and
one C-ABI call per current device does the work.  Token numbers and lengths are whole numbers in ordinary fp32 tensors,
exact up to 2^24.  A token below zero marks a padded place.  A number that is no row of the table, or no length, is taken
for padding and raises LnnError (E_INVALID) when a result is next read; what is queued meanwhile runs.
"""
from functools import lru_cache, partial

import numpy as np

from . import _lib
from . import deferred as _deferred
from . import ops
from .devices import devices
from .shape import TensorShape
from .tensor import Tensor

MAX_NUMBER = 1 << 24          # whole numbers that fp32 holds exactly
MAX_HEAD_DIM = 256

_call = _lib.call
_out = ops._out
_each_device = ops._each_device


def _tensors(names, *tensors):
    for name, t in zip(names.split(), tensors):
        if not isinstance(t, Tensor):
            raise ValueError(f"{name} must be a Tensor, got {t.__class__}")


@lru_cache(maxsize=4096)
def _shape(*dims):
    return TensorShape(dims)


def _whole(name, value, lowest):
    if not abs(value) < float("inf") or int(value) != value or value < lowest:
        raise ValueError(f"{name} {value} must be a whole number, at least {lowest}")
    return int(value)


# =============================================================================================
# embedding
# =============================================================================================
def embedding(ids_t, table_t, scale=1.0):
    """scale * table[ids]: ids of any shape, table (V, E) -> ids.shape + (E,).  Places with an id below zero are zero.

    The gradient of the table adds the terms of a row in the order of the tokens (they are sorted by row first), so that
    it is the same from run to run."""
    _tensors("ids_t table_t", ids_t, table_t)
    if table_t.shape.rank != 2:
        raise ValueError(f"table_t must be (tokens, dim), got {table_t.shape}")
    vocab, dim = table_t.shape.shape
    if vocab > MAX_NUMBER:
        raise ValueError(f"a table of {vocab} rows: token numbers are exact in fp32 up to {MAX_NUMBER}")
    scale = float(scale)
    n = ids_t.shape.size
    output_t = _out(_shape(*ids_t.shape.shape, dim), "embedding")

    def grad(O_t, dO_t):
        g, acc = table_t._grad_to_write()
        for i, dev in _each_device():
            _call.lnn_embedding_bwd_acc(i, dev, g, dO_t, ids_t, n, vocab, dim, scale, acc)

    output_t._assign_gradfn(table_t, grad)
    for i, dev in _each_device():
        _call.lnn_embedding_fwd(i, dev, output_t, table_t, ids_t, n, vocab, dim, scale)
    return output_t


# =============================================================================================
# probabilities of tokens
# =============================================================================================
def _logit_rows(logits_t, names, *of_rows):
    """(rows, vocab, result shape) after the checks; of_rows: the tensors with one element per row, or None"""
    _tensors("logits_t " + names, logits_t, *of_rows)
    dims = logits_t.shape.shape
    if len(dims) < 2:
        raise ValueError(f"logits_t must be (..., vocabulary) of rank 2 or more, got {logits_t.shape}")
    vocab = dims[-1]
    if vocab > MAX_NUMBER:
        raise ValueError(f"a vocabulary of {vocab}: token numbers are exact in fp32 up to {MAX_NUMBER}")
    rows = logits_t.shape.size // vocab
    for name, t in zip(names.split(), of_rows):
        if t.shape.size != rows:
            raise ValueError(f"{name} must have {rows} elements, one per row of logits_t, got {t.shape}")
    return rows, vocab, _shape(*dims[:-1])


def _logit_grad(logits_t, ids_t, stats_t, rows, vocab, O_t, dO_t):
    g, acc = logits_t._grad_to_write()
    for i, dev in _each_device():
        _call.lnn_token_logit_bwd_acc(i, dev, g, logits_t, stats_t, ids_t, dO_t, rows, vocab, acc)


def token_log_prob(logits_t, ids_t):
    """log(softmax(logits)[id]) of each row, with the maximum subtracted: logits (..., V), one id per row -> (...).
    Rows with an id below zero give 0 and no gradient."""
    rows, vocab, shape = _logit_rows(logits_t, "ids_t", ids_t)
    output_t, stats_t = _out(shape, "token_log_prob"), _out(_shape(rows, 3))
    output_t._assign_gradfn(logits_t, partial(_logit_grad, logits_t, ids_t, stats_t, rows, vocab))
    for i, dev in _each_device():
        _call.lnn_token_log_prob_fwd(i, dev, output_t, stats_t, logits_t, ids_t, rows, vocab)
    return output_t


def policy_loss(logits_t, ids_t, old_t, advantage_t, ref_t=None, clip_low=0.2, clip_high=0.2, kl=0.0):
    """The clipped policy loss of each row, with an optional KL term against a reference policy:

        logp = log(softmax(logits)[id]),  r = exp(logp - old)
        loss = -min(r * advantage, clip(r, 1 - clip_low, 1 + clip_high) * advantage)
               + kl * (exp(ref - logp) - (ref - logp) - 1)

    logits (..., V) -> (...); ids, old, advantage and ref have one element per row.  old and ref are logarithms as
    token_log_prob gives them.  The gradient goes to the logits; the other arguments are constants.  Rows with an id
    below zero give 0 and no gradient."""
    if ref_t is None:
        rows, vocab, shape = _logit_rows(logits_t, "ids_t old_t advantage_t", ids_t, old_t, advantage_t)
    else:
        rows, vocab, shape = _logit_rows(logits_t, "ids_t old_t advantage_t ref_t", ids_t, old_t, advantage_t, ref_t)
    clip_low, clip_high, kl = float(clip_low), float(clip_high), float(kl)
    if not 0.0 <= clip_low <= 1.0 or not 0.0 <= clip_high < float("inf"):
        raise ValueError(f"the ratio cannot be clipped to 1 - {clip_low} .. 1 + {clip_high}")
    if not 0.0 <= kl < float("inf"):
        raise ValueError(f"kl {kl} must not be negative")
    if kl != 0.0 and ref_t is None:
        raise ValueError("a KL term needs ref_t")
    if kl == 0.0:
        ref_t = None
    output_t, stats_t = _out(shape, "policy_loss"), _out(_shape(rows, 3))
    output_t._assign_gradfn(logits_t, partial(_logit_grad, logits_t, ids_t, stats_t, rows, vocab))
    for i, dev in _each_device():
        _call.lnn_policy_loss_fwd(i, dev, output_t, stats_t, logits_t, ids_t, old_t, advantage_t, ref_t, rows, vocab,
                                  clip_low, clip_high, kl)
    return output_t


# =============================================================================================
# attention
# =============================================================================================
_geom = lru_cache(maxsize=4096)(_lib.AttnGeom)           # (read only)


def _span(window, sinks):
    return _whole("window", window, 1), _whole("sinks", sinks, 0)


def _scale(scale, dim):
    if not 0 < dim <= MAX_HEAD_DIM:
        raise ValueError(f"heads of {dim} values: at most {MAX_HEAD_DIM}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) < float("inf"):
        raise ValueError(f"scale {scale} must be finite")
    return scale


class _AttentionGrad(_deferred.JointGrad):
    """Grad functions of queries, keys and values, which are wanted together."""

    def __init__(self, q_t, k_t, v_t, lengths_t, lse_t, geom):
        self.roles = (q_t, k_t, v_t)
        self.lengths_t, self.lse_t, self.geom = lengths_t, lse_t, geom
        self[q_t], self[k_t], self[v_t] = [], [], []

    def joint(self, O_t, dO_t, inputs):
        targets, flags, later, seen = [], [], [], set()
        for t in self.roles:
            source = t._get_top_reference_source()
            if not any(t is x for x in inputs):
                target, acc = None, 0
            elif source in seen:                        # one tensor in two places: its second gradient is added behind
                target, acc = _out(t.shape), 0
                later.append((t, target))
            else:
                target, acc = t._grad_to_write()
                seen.add(source)
            targets.append(target)
            flags.append(acc)
        q_t, k_t, v_t = self.roles
        for i, dev in _each_device():
            for target, acc in zip(targets, flags):
                if acc:
                    target._ptr(i)                      # (zero-filled where only another device's memory has been touched)
            _call.lnn_sink_attn_bwd(i, dev, *targets, q_t, k_t, v_t, O_t, self.lse_t, self.lengths_t, dO_t, self.geom.address,
                                    *flags)
        for t, extra in later:
            g = t.get_grad()
            ops.add_op(g, extra, output_t=g)
        for t in inputs:                                # those somebody has registered besides
            for func in self[t]:
                func(O_t, dO_t)


def sink_attention(q_t, k_t, v_t, window, sinks=0, scale=None, lengths_t=None):
    """Causal attention with a sliding window and `sinks` first tokens that stay visible.

    q (B, Hq, T, D), k and v (B, Hkv, S, D) -> (B, Hq, T, D); Hq is a multiple of Hkv (query heads share key heads in
    groups), T <= S, D <= 256.  Query i is at position p = i + S - T of its sequence and sees key j when j <= p and
    (p - j < window or j < sinks).  scale is D ** -0.5 unless given.  lengths_t, of B elements, says how many of the S
    keys of each sequence are real: the rest is padding behind it, whose rows give zeros and neither get nor pass on a
    gradient.  All three inputs have gradients."""
    _tensors("q_t k_t v_t", q_t, k_t, v_t)
    q_dims, k_dims = q_t.shape.shape, k_t.shape.shape
    if len(q_dims) != 4 or len(k_dims) != 4 or v_t.shape.shape != k_dims:
        raise ValueError(f"expected q (B, Hq, T, D) and k, v (B, Hkv, S, D), got {q_t.shape}, {k_t.shape}, {v_t.shape}")
    B, Hq, T, D = q_dims
    Hkv, S = k_dims[1], k_dims[2]
    if k_dims[0] != B or k_dims[3] != D or Hq % Hkv != 0:
        raise ValueError(f"q {q_t.shape} does not go with k and v {k_t.shape}")
    if T > S:
        raise ValueError(f"{T} queries over {S} keys: the last key belongs to the last query")
    if S > MAX_NUMBER:
        raise ValueError(f"{S} keys: lengths are exact in fp32 up to {MAX_NUMBER}")
    window, sinks = _span(window, sinks)
    scale = _scale(scale, D)
    if lengths_t is not None:
        _tensors("lengths_t", lengths_t)
        if lengths_t.shape.size != B:
            raise ValueError(f"lengths_t must have {B} elements, one per sequence, got {lengths_t.shape}")
    geom = _geom(B, Hq, Hkv, T, S, D, min(window, S), min(sinks, S), scale)
    output_t, lse_t = _out(q_t.shape, "sink_attention"), _out(_shape(B, Hq, T, 2))
    output_t._gradfns = _AttentionGrad(q_t, k_t, v_t, lengths_t, lse_t, geom)
    for i, dev in _each_device():
        _call.lnn_sink_attn_fwd(i, dev, output_t, lse_t, q_t, k_t, v_t, lengths_t, geom.address)
    return output_t


class SinkCache:
    """SinkCache(batch, heads, window, sinks, dim): keys and values of the positions that sink_attention sees from the end
    of each sequence, for sink_attention_step.

    k, v: tensors (batch, heads, sinks + window, dim).  Position p is in slot p (p < sinks) or
    sinks + (p - sinks) % window.  lengths: tensor (batch,), how many positions each sequence has seen, 0 at first and
    at most 2^24; below zero, the place in the batch is not in use.  (A step writes its lengths to another tensor:
    ask for `lengths` after it.)"""

    def __init__(self, batch, heads, window, sinks, dim):
        self.batch, self.heads = _whole("batch", batch, 1), _whole("heads", heads, 1)
        self.window, self.sinks = _span(window, sinks)
        self.dim = _whole("dim", dim, 1)
        _scale(None, self.dim)
        if self.window + self.sinks > MAX_NUMBER:
            raise ValueError(f"{self.window + self.sinks} slots: at most {MAX_NUMBER}")
        shape = (self.batch, self.heads, self.sinks + self.window, self.dim)
        self._token_shape = (self.batch, self.heads, self.dim)
        self.k, self.v = Tensor(shape), Tensor(shape)
        self._lengths = [Tensor((self.batch,)), Tensor((self.batch,))]

    @property
    def lengths(self):
        return self._lengths[0]

    def set_lengths(self, value):
        """A tensor, array or list of `batch` whole numbers, or one number for all."""
        if not isinstance(value, Tensor):
            value = np.asarray(value, np.float32)
            if value.ndim == 0:
                value = np.full(self.batch, value)
        if (value.shape.size if isinstance(value, Tensor) else value.size) != self.batch:
            raise ValueError(f"lengths must have {self.batch} elements")
        if not isinstance(value, Tensor):
            value = value.reshape(self.batch)
        self.lengths.set(value)

    def store(self, k_t, v_t, lengths_t=None):
        """Fill the cache from a prompt: k and v (batch, heads, S, dim), of which lengths_t (S everywhere unless given) are
        real.  Slots that no position of the prompt falls into stay as they are, and so does the place of a sequence
        whose length is below zero."""
        _tensors("k_t v_t", k_t, v_t)
        dims = k_t.shape.shape
        if len(dims) != 4 or v_t.shape.shape != dims or (dims[0], dims[1], dims[3]) != self._token_shape:
            raise ValueError(f"expected k and v ({self.batch}, {self.heads}, S, {self.dim}), got {k_t.shape}, {v_t.shape}")
        S = dims[2]
        if S > MAX_NUMBER:
            raise ValueError(f"{S} keys: lengths are exact in fp32 up to {MAX_NUMBER}")
        if lengths_t is not None:
            _tensors("lengths_t", lengths_t)
            if lengths_t.shape.size != self.batch:
                raise ValueError(f"lengths_t must have {self.batch} elements, one per sequence, got {lengths_t.shape}")
        sources = [t._get_top_reference_source() for t in (k_t, v_t, lengths_t) if t is not None]
        if any(s is t for s in sources for t in (self.k, self.v, self.lengths)):
            raise ValueError("the cache cannot be filled from itself")
        for i, dev in _each_device():
            _call.lnn_sink_cache_store(i, dev, self.k, self.v, self.lengths, k_t, v_t, lengths_t, self.batch, self.heads, S,
                                       self.dim, self.window, self.sinks)


def sink_attention_step(q_t, k_t, v_t, cache, scale=None):
    """One more token of each sequence: its key and value (batch, heads, dim) go into the cache, and its query
    (batch, Hq, dim) attends over what sink_attention would see -> (batch, Hq, dim).  Hq is a multiple of the cache's
    heads.  Places of a length below zero give zeros and stay as they are.  Forward only: no grad functions."""
    _tensors("q_t k_t v_t", q_t, k_t, v_t)
    if not isinstance(cache, SinkCache):
        raise ValueError(f"cache must be a SinkCache, got {cache.__class__}")
    dims = q_t.shape.shape
    if k_t.shape.shape != cache._token_shape or v_t.shape.shape != cache._token_shape:
        raise ValueError(f"expected k and v {cache._token_shape}, got {k_t.shape}, {v_t.shape}")
    if len(dims) != 3 or dims[0] != cache.batch or dims[2] != cache.dim or dims[1] % cache.heads != 0:
        raise ValueError(f"q {q_t.shape} does not go with a cache of {cache._token_shape}")
    for t in (q_t, k_t, v_t):
        source = t._get_top_reference_source()
        if source is cache.k or source is cache.v:
            raise ValueError("the token cannot be part of the cache's own memory")
    scale = _scale(scale, cache.dim)
    output_t = _out(q_t.shape, "sink_attention_step")
    now, after = cache._lengths
    for i, dev in _each_device():
        _call.lnn_sink_attn_step(i, dev, output_t, q_t, k_t, v_t, cache.k, cache.v, now, after, cache.batch, dims[1],
                                 cache.heads, cache.dim, cache.window, cache.sinks, scale)
    if devices._shallow == 0:
        cache._lengths = [after, now]
    return output_t
