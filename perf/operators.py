"""The operators on tokens as cases to be timed: what a program that trains or serves a sequence model asks of them.

Five kinds, each with a range that `draw` samples and that the listed cases stand for:

  embed    rows of a table for a batch of tokens; with `train` the gradient of the table too
  prompt   attention over a prompt with a sliding window and a few first tokens that stay visible, and the
           cache that the answer goes on from
  attend   the same attention in training: forward and the gradients of queries, keys and values
  step     one more token per sequence: appended to that cache, and attention over it
  policy   the logarithm of the chosen tokens' probabilities; with `train` the clipped policy loss with a KL
           term and the gradient of the logits

Tensors are fp32, as everywhere in the framework; token numbers and lengths are whole numbers in fp32 tensors, and a
token below zero marks a padded place.
"""
import functools
import math

import torch

own = False


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # the token a server has just chosen
        {"name": "embed_1", "kind": "embed", "tokens": 1, "vocab": 32768, "dim": 1024, "train": False},
        # a training batch of natural text: the most frequent token is some thousand times in it
        {"name": "embed_16384_train", "kind": "embed", "tokens": 16384, "vocab": 50001, "dim": 768, "train": True},
        # a short question: launch latency
        {"name": "prompt_37", "kind": "prompt", "batch": 1, "heads": 4, "kv_heads": 4, "new": 37, "past": 0, "dim": 64,
         "window": 256, "sinks": 4, "ragged": False},
        # a long document
        {"name": "prompt_8192", "kind": "prompt", "batch": 1, "heads": 16, "kv_heads": 4, "new": 8192, "past": 0, "dim": 128,
         "window": 1024, "sinks": 4, "ragged": False},
        # a batch of examples of unequal length, extents that no tile divides
        {"name": "attend_4x777", "kind": "attend", "batch": 4, "heads": 6, "kv_heads": 6, "new": 777, "past": 0, "dim": 80,
         "window": 200, "sinks": 3, "ragged": True},
        # long examples, shared key and value heads
        {"name": "attend_8192", "kind": "attend", "batch": 1, "heads": 8, "kv_heads": 2, "new": 8192, "past": 0, "dim": 128,
         "window": 2048, "sinks": 16, "ragged": False},
        # one conversation
        {"name": "step_1", "kind": "step", "batch": 1, "heads": 8, "kv_heads": 2, "dim": 64, "window": 1020, "sinks": 4},
        # a full server
        {"name": "step_64", "kind": "step", "batch": 64, "heads": 32, "kv_heads": 8, "dim": 128, "window": 4092, "sinks": 4},
        # the tokens of a few answers are scored under the policy that gave them
        {"name": "score_64", "kind": "policy", "tokens": 64, "vocab": 131072, "train": False},
        # scoring a whole batch, an odd vocabulary: rows start at any 4-byte boundary
        {"name": "score_4096", "kind": "policy", "tokens": 4096, "vocab": 32003, "train": False},
        # a toy policy, launch latency
        {"name": "policy_37", "kind": "policy", "tokens": 37, "vocab": 1003, "train": True},
        # a training step's answers
        {"name": "policy_2048", "kind": "policy", "tokens": 2048, "vocab": 131072, "train": True},
    ]


def _log(rng, lo, hi):
    """A whole number whose logarithm is uniform between lo and hi."""
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["embed", "prompt", "attend", "step", "policy"])
    if kind == "embed":
        return {"kind": kind, "tokens": _log(rng, 1, 32768), "vocab": _log(rng, 64, 65536), "dim": _log(rng, 16, 1024),
                "train": rng.random() < 0.6}
    if kind == "policy":
        vocab = _log(rng, 256, 131072)
        return {"kind": kind, "tokens": _log(rng, 1, min(8192, (1 << 28) // vocab)), "vocab": vocab, "train": rng.random() < 0.6}
    kv_heads = rng.choice([1, 2, 2, 3, 4, 8])
    case = {"kind": kind, "batch": 1, "heads": kv_heads * rng.choice([1, 1, 2, 4]), "kv_heads": kv_heads}
    if kind == "step":
        case["batch"] = _log(rng, 1, 64)
        return dict(case, dim=rng.choice([32, 64, 64, 80, 128, 128]), window=_log(rng, 16, 4096),
                    sinks=rng.choice([0, 1, 4, 4, rng.randint(2, 64)]))
    case["batch"] = rng.choice([1, 1, 2, rng.randint(2, 8)])
    # the plain form holds all pairs of positions
    top = math.isqrt((16 if kind == "prompt" else 8) * 8192 * 8192 // (case["batch"] * case["heads"]))
    new = _log(rng, 1 if kind == "prompt" else 16, min(8192, top))
    past = rng.choice([0, 0, _log(rng, 1, 1024)]) if new < min(8192, top) - 1024 else 0
    return dict(case, new=new, past=past, dim=rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128]),
                window=_log(rng, 2, 4096), sinks=rng.choice([0, 1, 4, 4, rng.randint(2, 64)]),
                ragged=case["batch"] > 1 and rng.random() < 0.5)


def _lengths(case):
    """How many of the keys of each sequence are real."""
    n, b = case["new"] + case["past"], case["batch"]
    return [n - i * n // (2 * b) if case["ragged"] else n for i in range(b)]


# ---------------------------------------------------------------------------------------------
# preparation: what a program holds before the call
# ---------------------------------------------------------------------------------------------
class _Memory:
    def __init__(self, pointer, shape):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": "<f4", "data": (pointer, False), "version": 3}


@functools.lru_cache(maxsize=4096)
def _view(pointer, shape):
    """The framework's memory as torch sees it.  It holds an address and no values; a user's program has no need of it."""
    return torch.as_tensor(_Memory(pointer, shape), device="cuda:0")


class _Result(list):
    """Outputs of a pass as torch tensors over the framework's own buffers; keeps them alive."""
    owners = ()


def _outputs(*tensors):
    r = _Result(_view(t._ptr(0), t.shape.shape) for t in tensors)
    r.owners = tensors
    return r


def _inputs(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (lambda *shape: torch.randn(shape, generator=g, device="cuda"),
            lambda *shape: torch.rand(shape, generator=g, device="cuda"))


def _values(case, seed):
    """Inputs of a case as torch tensors."""
    normal, uniform = _inputs(seed)
    kind = case["kind"]
    if kind == "embed":
        n, v, e = case["tokens"], case["vocab"], case["dim"]
        # word frequencies fall as one over the rank; one place of 16 is padding
        ids = (torch.exp(uniform(n) * math.log(v)) - 1).floor().clamp(0, v - 1)
        if n > 16:
            ids[-(n // 16):] = -1
        return {"ids": ids, "table": normal(v, e) * 0.02, "dy": normal(n, e) * 0.1}
    if kind == "policy":
        n, v = case["tokens"], case["vocab"]
        z = normal(n, v) * 2.5
        ids = (z - torch.log(-torch.log(uniform(n, v).clamp(1e-7, 1 - 1e-6)))).argmax(1)       # sampled from the policy
        logp = (z.gather(1, ids[:, None])[:, 0] - torch.logsumexp(z, 1))
        ids = ids.float()
        if n > 16:
            ids[-(n // 16):] = -1
        old = logp + 0.15 * normal(n)
        return {"logits": z, "ids": ids, "old": old, "ref": old + 0.1 * normal(n), "adv": normal(n),
                "dy": torch.full((n,), 1.0 / n, device="cuda")}
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if kind == "step":
        cap = case["window"] + case["sinks"]
        return {"q": normal(b, h, d), "k": normal(b, hk, d), "v": normal(b, hk, d), "cache_k": normal(b, hk, cap, d),
                "cache_v": normal(b, hk, cap, d), "lengths": (cap + uniform(b) * 3 * cap).floor()}
    s = case["new"] + case["past"]
    x = {"q": normal(b, h, case["new"], d), "k": normal(b, hk, s, d), "v": normal(b, hk, s, d),
         "lengths": torch.tensor(_lengths(case), dtype=torch.float32, device="cuda")}
    if kind == "attend":
        x["dy"] = normal(b, h, case["new"], d) * 0.1
    return x


def prepare(case, seed):
    s = _values(case, seed)
    if case["kind"] == "prompt":
        shape = (case["batch"], case["kv_heads"], case["window"] + case["sinks"], case["dim"])
        s["cache_k"], s["cache_v"] = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    if own:
        # a program written for the framework has its tensors, its cache and its optimizer in hand
        import litenn_b200 as nn
        torch.cuda.synchronize()
        for name, x in s.items():
            if not name.startswith("cache"):
                t = nn.Tensor(tuple(x.shape))
                _view(t._ptr(0), tuple(x.shape)).copy_(x)
                s[name] = t
        if case["kind"] in ("prompt", "step"):
            s["cache"] = nn.SinkCache(case["batch"], case["kv_heads"], case["window"], case["sinks"], case["dim"])
            if case["kind"] == "step":
                for t, x in ((s["cache"].k, s["cache_k"]), (s["cache"].v, s["cache_v"])):
                    _view(t._ptr(0), tuple(x.shape)).copy_(x)
                s["cache"].set_lengths(s["lengths"])
            del s["cache_k"], s["cache_v"]
        leaves = {"embed": ["table"], "attend": ["q", "k", "v"], "policy": ["logits"]}.get(case["kind"])
        if leaves and case.get("train", True):
            s["opt"] = nn.optimizer.SGD([s[name] for name in leaves])       # makes them trainable; no step is taken
        torch.cuda.synchronize()
    s["case"] = case
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
SCALE = 27.7          # of the embedding
CLIP, KL = 0.2, 0.05


def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state, state["case"])


def _plain_embed(s, c):
    ids, table = s["ids"].long(), s["table"]
    real = (ids >= 0)[:, None]
    at = ids.clamp(min=0)
    y = torch.where(real, table[at] * SCALE, 0.0)
    if not c["train"]:
        return [y]
    dy = torch.where(real, s["dy"].double() * SCALE, 0.0)          # a frequent token's sum is long
    return [y, torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, at, dy).float()]


def _mask(c, lengths, device):
    at = torch.arange(c["new"], device=device)[:, None] + c["past"]
    key = torch.arange(c["new"] + c["past"], device=device)[None, :]
    seen = (key <= at) & ((at - key < c["window"]) | (key < c["sinks"]))
    return (seen[None] & (at[None] < lengths.long()[:, None, None]))[:, None, None]


def _plain_attention(s, c):
    """(output, probabilities, queries, keys and values in groups of heads that share a key head)"""
    b, hk, t, d = c["batch"], c["kv_heads"], c["new"], c["dim"]
    q = s["q"].reshape(b, hk, c["heads"] // hk, t, d)
    k, v = s["k"][:, :, None], s["v"][:, :, None]
    x = torch.where(_mask(c, s["lengths"], q.device), (q * d ** -0.5) @ k.transpose(-1, -2), -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return p @ v, p, q, k, v


def _plain_prompt(s, c):
    o = _plain_attention(s, c)[0].reshape(s["q"].shape)
    # the slot of position p: the first ones keep theirs, the others go round
    sinks, window = c["sinks"], c["window"]
    slot = torch.arange(sinks + window, device=o.device)[None, :]
    last = s["lengths"].long()[:, None] - 1
    ring = slot - sinks + (last - slot).div(window, rounding_mode="floor") * window + sinks
    at = torch.where(slot < sinks, slot, ring)
    filled = ((at >= slot) & (at <= last))[:, None, :, None]
    at = at.clamp(0, c["new"] + c["past"] - 1)[:, None, :, None].expand(s["cache_k"].shape)
    s["cache_k"] = torch.where(filled, s["k"].gather(2, at), s["cache_k"])
    s["cache_v"] = torch.where(filled, s["v"].gather(2, at), s["cache_v"])
    return [o, s["cache_k"], s["cache_v"]]


def _plain_attend(s, c):
    o, p, q, k, v = _plain_attention(s, c)
    do = s["dy"].reshape(o.shape)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v.transpose(-1, -2) - (do * o).sum(-1, keepdim=True)) * c["dim"] ** -0.5
    return [o.reshape(s["q"].shape), (ds @ k).reshape(s["q"].shape), (ds.transpose(-1, -2) @ q).sum(2), dv]


def _plain_step(s, c):
    b, h, hk, d, sinks, window = (c[x] for x in ("batch", "heads", "kv_heads", "dim", "sinks", "window"))
    n = s["lengths"].long()
    slot = torch.where(n < sinks, n, sinks + (n - sinks) % window)
    rows = torch.arange(b, device=n.device)
    s["cache_k"][rows, :, slot] = s["k"]
    s["cache_v"][rows, :, slot] = s["v"]
    s["lengths"] = s["lengths"] + 1
    x = (s["q"].reshape(b, hk, h // hk, d) * d ** -0.5) @ s["cache_k"].transpose(-1, -2)
    full = torch.arange(sinks + window, device=n.device)[None, :] <= n[:, None]
    x = torch.where(full[:, None, None], x, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    o = (e / e.sum(-1, keepdim=True)) @ s["cache_v"]
    return [o.reshape(b, h, d), s["cache_k"], s["cache_v"], s["lengths"]]


def _plain_policy(s, c):
    # in 64 bits: whether a ratio is clipped is decided next to a border
    z, ids = s["logits"], s["ids"].long()
    real, at = ids >= 0, ids.clamp(min=0)[:, None]
    top = z.amax(1, keepdim=True)
    e = torch.exp((z - top).double())
    total = e.sum(1, keepdim=True)
    logp = (z.gather(1, at) - top).double()[:, 0] - torch.log(total)[:, 0]
    if not c["train"]:
        return [torch.where(real, logp, 0.0).float()]
    old, ref, adv = s["old"].double(), s["ref"].double(), s["adv"].double()
    r, u = torch.exp(logp - old), ref - logp
    loss = -torch.minimum(r * adv, r.clamp(1 - CLIP, 1 + CLIP) * adv) + KL * (torch.exp(u) - u - 1)
    inside = torch.where(adv >= 0, r <= 1 + CLIP, r >= 1 - CLIP)
    slope = torch.where(inside, -adv * r, 0.0) + KL * (1 - torch.exp(u))
    slope = torch.where(real, slope * s["dy"], 0.0)[:, None]
    dz = e * (-slope / total)
    dz.scatter_add_(1, at, slope)
    return [torch.where(real, loss, 0.0).float(), dz.float()]


def _own_embed(s, c):
    import litenn_b200 as nn
    if not c["train"]:
        return _outputs(nn.embedding(s["ids"], s["table"], SCALE))
    s["opt"].zero_grad()
    y = nn.embedding(s["ids"], s["table"], SCALE)
    nn.backward({y: s["dy"]})
    return _outputs(y, s["table"].get_grad())


def _own_prompt(s, c):
    import litenn_b200 as nn
    o = nn.sink_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"], lengths_t=s["lengths"])
    s["cache"].store(s["k"], s["v"], lengths_t=s["lengths"])
    return _outputs(o, s["cache"].k, s["cache"].v)


def _own_attend(s, c):
    import litenn_b200 as nn
    s["opt"].zero_grad()
    o = nn.sink_attention(s["q"], s["k"], s["v"], c["window"], c["sinks"], lengths_t=s["lengths"])
    nn.backward({o: s["dy"]})
    return _outputs(o, s["q"].get_grad(), s["k"].get_grad(), s["v"].get_grad())


def _own_step(s, c):
    import litenn_b200 as nn
    o = nn.sink_attention_step(s["q"], s["k"], s["v"], s["cache"])
    return _outputs(o, s["cache"].k, s["cache"].v, s["cache"].lengths)


def _own_policy(s, c):
    import litenn_b200 as nn
    if not c["train"]:
        return _outputs(nn.token_log_prob(s["logits"], s["ids"]))
    s["opt"].zero_grad()
    loss = nn.policy_loss(s["logits"], s["ids"], s["old"], s["adv"], ref_t=s["ref"], clip_low=CLIP, clip_high=CLIP, kl=KL)
    nn.backward({loss: s["dy"]})
    return _outputs(loss, s["logits"].get_grad())


_plain = {"embed": _plain_embed, "prompt": _plain_prompt, "attend": _plain_attend, "step": _plain_step, "policy": _plain_policy}
_own = {"embed": _own_embed, "prompt": _own_prompt, "attend": _own_attend, "step": _own_step, "policy": _own_policy}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_attention(q, k, v, seen):
    """softmax over what each row sees; rows that see nothing are zero"""
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    x = torch.einsum("bhid,bhjd->bhij", q, k) / math.sqrt(q.shape[-1])
    x = x.masked_fill(~seen, -math.inf).masked_fill(~seen.any(-1, keepdim=True), 0.0)
    return torch.einsum("bhij,bhjd->bhid", torch.softmax(x, -1) * seen.any(-1, keepdim=True), v)


def exact(case, seed):
    x, kind = _values(case, seed), case["kind"]
    w = {n: t.double() for n, t in x.items()}
    if kind == "embed":
        ids, e = x["ids"].long(), case["dim"]
        padded = torch.cat([w["table"], torch.zeros(1, e, dtype=torch.float64, device="cuda")])
        padded.requires_grad_(True)
        y = padded[torch.where(ids < 0, case["vocab"], ids)] * SCALE
        if not case["train"]:
            return [y.detach()]
        index = torch.where(ids < 0, case["vocab"], ids)[:, None].expand(-1, e)
        return [y.detach(), torch.zeros_like(padded).scatter_add(0, index, w["dy"])[:-1].detach() * SCALE]
    if kind == "policy":
        z = w["logits"].requires_grad_(case["train"])
        real = (x["ids"] >= 0).double()
        logp = torch.log_softmax(z, 1)[torch.arange(len(real), device="cuda"), x["ids"].long().clamp(min=0)]
        if not case["train"]:
            return [logp * real]
        r = (logp - w["old"]).exp()
        gain = torch.where(w["adv"] >= 0, r.clamp(max=1 + CLIP), r.clamp(min=1 - CLIP)) * w["adv"]
        loss = (KL * ((w["ref"] - logp).exp() + logp - w["ref"] - 1) - gain) * real
        (loss * w["dy"]).sum().backward()
        return [loss.detach(), z.grad]
    if kind == "step":
        sinks, window = case["sinks"], case["window"]
        for b, n in enumerate(int(n) for n in x["lengths"].tolist()):
            slot = n if n < sinks else (n - sinks) % window + sinks
            w["cache_k"][b, :, slot], w["cache_v"][b, :, slot] = w["k"][b], w["v"][b]
        seen = (torch.arange(sinks + window, device="cuda")[None] <= w["lengths"][:, None])[:, None, None]
        o = _exact_attention(w["q"][:, :, None], w["cache_k"], w["cache_v"], seen)[:, :, 0]
        return [o, w["cache_k"], w["cache_v"], w["lengths"] + 1]
    i = torch.arange(case["past"], case["past"] + case["new"], device="cuda")
    j = torch.arange(case["past"] + case["new"], device="cuda")
    back = i[:, None] - j[None]
    seen = (back >= 0) & ((back < case["window"]) | (j < case["sinks"]))
    seen = seen[None, None] & (i[:, None] < w["lengths"][:, None, None, None])
    leaves = [w[n].requires_grad_(kind == "attend") for n in ("q", "k", "v")]
    o = _exact_attention(*leaves, seen)
    if kind == "attend":
        o.backward(w["dy"])
        return [o.detach()] + [t.grad for t in leaves]
    caches = []
    for t in (w["k"], w["v"]):
        cache = torch.zeros(*t.shape[:2], case["sinks"] + case["window"], case["dim"], dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(case)):
            first, ring = min(n, case["sinks"]), torch.arange(max(case["sinks"], n - case["window"]), n, device="cuda")
            cache[b, :, :first] = t[b, :, :first]
            if len(ring):
                cache[b, :, case["sinks"] + (ring - case["sinks"]) % case["window"]] = t[b, :, ring]
        caches.append(cache)
    return [o, *caches]


# ---------------------------------------------------------------------------------------------
# the work of a pass
# ---------------------------------------------------------------------------------------------
def _pairs(case):
    """Visible pairs of a query and a key, over the batch, for one head."""
    w, n = case["window"], 0
    for length in _lengths(case):
        lo, hi = case["past"], min(case["past"] + case["new"], length)      # positions of the queries that see anything
        if hi > lo:
            full = max(0, hi - max(lo, w))                                  # those whose window is full
            some = range(lo, min(hi, w))
            n += full * w + (some[0] + 1 + some[-1] + 1) * len(some) // 2 if len(some) else full * w
            # first tokens in front of the window: min(sinks, p + 1 - w)
            n += sum(min(case["sinks"], p + 1 - w) for p in range(max(lo, w), min(hi, w + case["sinks"])))
            n += max(0, hi - max(lo, w + case["sinks"])) * case["sinks"]
    return n


def work(case):
    kind = case["kind"]
    if kind == "embed":
        n, e = case["tokens"], case["dim"]
        if not case["train"]:
            return {"bytes": 4 * (n + 2 * n * e), "flops": n * e}
        return {"bytes": 4 * (n + 3 * n * e + case["vocab"] * e), "flops": 3 * n * e}
    if kind == "policy":
        n, v = case["tokens"], case["vocab"]
        if not case["train"]:
            return {"bytes": 4 * (n * v + 2 * n), "flops": 4 * n * v}
        return {"bytes": 4 * (2 * n * v + 6 * n), "flops": 7 * n * v}
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if kind == "step":
        n = case["window"] + case["sinks"]
        return {"bytes": 4 * (2 * b * hk * n * d + 2 * b * h * d + 4 * b * hk * d), "flops": 4 * b * h * n * d}
    q, k, pairs = b * h * case["new"] * d, b * hk * (case["new"] + case["past"]) * d, h * _pairs(case)
    if kind == "prompt":
        cache = b * hk * min(case["new"] + case["past"], case["window"] + case["sinks"]) * d
        return {"bytes": 4 * (2 * q + 2 * k + 2 * cache), "flops": 4 * d * pairs}
    return {"bytes": 4 * (4 * q + 4 * k), "flops": 14 * d * pairs}
