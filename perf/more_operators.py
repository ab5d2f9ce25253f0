"""Attention with shaped scores, its form over a paged cache, and the clip by the joint norm, as
measurable cases.

A decoder is trained with attention whose scores are capped by a tanh, lowered with the distance of
query and key, or closed by documents packed into one row, by padding and by a prefix that all may
see; its gradients are clipped by their joint norm; and it then answers a few tokens at a time over
pages that hold the keys and values of what came before.

Tensors of this framework live in host memory between calls, so a case's pass is a whole call: its
inputs go to the device, the step loop runs there, and what it returns comes back. Training and
generation take as many steps as put the device's work above the transfers; what comes back is the
state at the end and the last gradients, as a training or serving program keeps them.

Kinds of work (a case's `kind`):
- attend: gradient descent on the queries, keys, values and slopes of one attention, as a layer
  inside a model meets it, `steps` steps in one run.
- cached: new tokens read over a paged cache and appended to it, `steps` times, each from the last
  one's result; one token a step or a chunk of a prompt.
- clip: descent on the parameters of a small decoder, their gradients clipped by the joint norm.
"""

import math

import numpy as np
import torch

own = False

_DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
_RATE = 0.05


def listed():
    return [
        # Attention inside a small model being trained, heads of a fused projection, capped scores.
        {"name": "attend cap 2x2048x8x64", "kind": "attend", "batch": 2, "length": 2048, "heads": 8, "keys": 8, "head": 64, "joined": True,
         "causal": True, "cap": 20.0, "slopes": False, "documents": 0, "prefix": False, "ragged": False, "dtype": "float32", "steps": 12},
        # Documents packed into rows of one length, grouped heads, a bias that falls with distance.
        {"name": "attend packed 4x1024x8x64", "kind": "attend", "batch": 4, "length": 1024, "heads": 8, "keys": 2, "head": 64, "joined": True,
         "causal": True, "cap": 0.0, "slopes": True, "documents": 5, "prefix": False, "ragged": False, "dtype": "float32", "steps": 24},
        # Prefixes that every token sees, a padded batch, odd sizes.
        {"name": "attend prefix 3x777x6x44", "kind": "attend", "batch": 3, "length": 777, "heads": 6, "keys": 3, "head": 44, "joined": False,
         "causal": True, "cap": 8.0, "slopes": False, "documents": 0, "prefix": True, "ragged": True, "dtype": "float32", "steps": 24},
        # Double precision, as used where gradients are checked, everything at once.
        {"name": "attend f64 2x130x4x32", "kind": "attend", "batch": 2, "length": 130, "heads": 4, "keys": 2, "head": 32, "joined": False,
         "causal": True, "cap": 10.0, "slopes": True, "documents": 3, "prefix": True, "ragged": True, "dtype": "float64", "steps": 24},
        # A short context: the time of the launches.
        {"name": "attend short 2x40x4x32", "kind": "attend", "batch": 2, "length": 40, "heads": 4, "keys": 4, "head": 32, "joined": True,
         "causal": True, "cap": 0.0, "slopes": True, "documents": 0, "prefix": False, "ragged": False, "dtype": "float32", "steps": 128},
        # One long text, wide heads.
        {"name": "attend long 1x5000x4x128", "kind": "attend", "batch": 1, "length": 5000, "heads": 4, "keys": 4, "head": 128, "joined": True,
         "causal": True, "cap": 30.0, "slopes": False, "documents": 0, "prefix": False, "ragged": False, "dtype": "float32", "steps": 6},
        # Sixteen conversations of several lengths, one token a step.
        {"name": "tokens 16x2048x8x64", "kind": "cached", "batch": 16, "length": 1, "heads": 8, "keys": 2, "head": 64, "past": 2048, "page": 64,
         "cap": 20.0, "slopes": False, "ragged": False, "dtype": "float32", "steps": 512},
        # One long conversation, one token a step: few heads over a long axis.
        {"name": "tokens 1x60000x8x64", "kind": "cached", "batch": 1, "length": 1, "heads": 8, "keys": 2, "head": 64, "past": 60000, "page": 256,
         "cap": 0.0, "slopes": True, "ragged": False, "dtype": "float32", "steps": 256},
        # Chunks of four prompts, wide heads.
        {"name": "chunk 4x256x8x128", "kind": "cached", "batch": 4, "length": 256, "heads": 8, "keys": 2, "head": 128, "past": 2048, "page": 64,
         "cap": 30.0, "slopes": False, "ragged": False, "dtype": "float32", "steps": 8},
        # Few new tokens of several counts, pages that end inside a tile, double precision.
        {"name": "chunk f64 3x17x6x40", "kind": "cached", "batch": 3, "length": 17, "heads": 6, "keys": 2, "head": 40, "past": 333, "page": 24,
         "cap": 10.0, "slopes": True, "ragged": True, "dtype": "float64", "steps": 16},
        # The gradients of a small decoder.
        {"name": "clip 6x256", "kind": "clip", "layers": 6, "model": 256, "vocab": 96, "dtype": "float32", "steps": 100},
        # Odd sizes, double precision.
        {"name": "clip f64 3x37", "kind": "clip", "layers": 3, "model": 37, "vocab": 65, "dtype": "float64", "steps": 100},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "cached", "cached", "cached", "clip"])
    dtype = rng.choice(["float32", "float32", "float32", "float64"])
    if kind == "clip":
        return {"kind": kind, "layers": rng.randint(1, 6), "model": _log_int(rng, 8, 256), "vocab": rng.randint(30, 200), "dtype": dtype,
                "steps": rng.randint(16, 64)}
    keys, head = rng.randint(1, 4), rng.choice([16, 24, 32, 40, 44, 64, 64, 64, 80, 96, 128])
    heads = keys * rng.choice([1, 1, 2, 3, 4])
    case = {"kind": kind, "batch": rng.randint(1, 4), "heads": heads, "keys": keys, "head": head, "cap": rng.choice([0.0, 0.0, 5.0, 15.0, 30.0]),
            "slopes": rng.random() < 0.4, "ragged": rng.random() < 0.4, "dtype": dtype}
    wide = 2 if dtype == "float64" else 1
    if kind == "attend":
        most = int(math.sqrt(2 ** 25 / (wide * case["batch"] * heads)))
        return {**case, "length": _log_int(rng, 1, min(3000, most)), "joined": rng.random() < 0.5, "causal": rng.random() < 0.8,
                "documents": rng.choice([0, 0, 0, 2, 7]), "prefix": rng.random() < 0.3, "steps": rng.randint(6, 12)}
    length = rng.choice([1, 1, 1, rng.randint(2, 16), rng.randint(17, 200)])
    most = 2 ** 21 // (wide * case["batch"] * keys * head)
    return {**case, "length": length, "past": _log_int(rng, 16, max(64, min(8192, most))), "page": rng.choice([8, 16, 24, 64, 100, 256]),
            "steps": rng.randint(16, 64) if length == 1 else rng.randint(3, 8)}


# ---- inputs -------------------------------------------------------------------------------------

def _normal(gen, shape, std, dtype=np.float32):
    return (gen.standard_normal(shape, dtype=np.float32) * np.float32(std)).astype(dtype)


def _slopes(gen, heads, dtype):
    """Slopes from 1/2 down to 1/256, moved a little by training."""
    return (np.exp2(-8.0 * np.arange(1, heads + 1) / heads) * np.exp(0.1 * gen.standard_normal(heads))).astype(dtype)


def _documents(gen, batch, length, most):
    """Ids of documents packed one after the other, up to `most` of them in a row, and in the last
    row a tail that belongs to none."""
    ids = np.empty((batch, length), np.int32)
    for row in ids:
        ends = np.sort(gen.integers(0, length, int(gen.integers(1, most + 1)) - 1))
        row[:] = 10 + np.searchsorted(ends, np.arange(length), side="right")
    ids[-1, length - length // 8:] = -1
    return ids


def _heads(c):
    return c["heads"] + 2 * c["keys"]


def _shapes(c):
    """Shapes of a small decoder's parameters, by name."""
    d, shapes = c["model"], {"tok": (c["vocab"], c["model"]), "head": (c["model"], c["vocab"]), "gain": (c["model"],), "shift": (c["model"],)}
    for k in range(c["layers"]):
        shapes.update({f"l{k}_qkv": (d, 3 * d), f"l{k}_qkv_b": (3 * d,), f"l{k}_out": (d, d), f"l{k}_out_b": (d,), f"l{k}_fc1": (d, 4 * d),
                       f"l{k}_fc1_b": (4 * d,), f"l{k}_fc2": (4 * d, d), f"l{k}_fc2_b": (d,), f"l{k}_gain": (2, d), f"l{k}_shift": (2, d)})
    return shapes


def _pages_each(c):
    return -(-(c["past"] + c["steps"] * c["length"]) // c["page"])


def _inputs(c, seed):
    """(state, data) of a case as dicts of numpy arrays, from the seed alone. What is trained or
    carried from step to step is the state."""
    gen, dtype = np.random.default_rng(seed), np.dtype(c["dtype"])
    if c["kind"] == "clip":
        shapes = _shapes(c)
        return ({k: _normal(gen, s, 0.5, dtype) for k, s in sorted(shapes.items())}, {k: _normal(gen, s, 0.5, dtype) for k, s in sorted(shapes.items())})
    b, t, h, n, hd = c["batch"], c["length"], c["heads"], c["keys"], c["head"]
    data = {}
    if c["kind"] == "attend":
        if c["joined"]:
            state = {"x": _normal(gen, (b, t, h + 2 * n, hd), 1.2, dtype)}
        else:
            state = {"q": _normal(gen, (b, t, h, hd), 1.2, dtype), "k": _normal(gen, (b, t, n, hd), 1.2, dtype), "v": _normal(gen, (b, t, n, hd), 1.2, dtype)}
        if c["slopes"]:
            state["slopes"] = _slopes(gen, h, dtype)
        if c["documents"]:
            data["documents"] = _documents(gen, b, t, c["documents"])
        if c["prefix"]:
            data["prefix"] = gen.integers(0, t // 2 + 1, b).astype(np.int32)
        data["t"] = _normal(gen, (b, t, h, hd), 0.5, dtype)
        if c["ragged"]:
            lengths = gen.integers(1, t + 1, b).astype(np.int32)
            lengths[0] = t
            data["lengths"] = lengths
            data["t"] *= np.arange(t)[None, :, None, None] < lengths[:, None, None, None]
        return state, data
    each = _pages_each(c)
    pages = b * each + 3  # a few belong to nobody
    state = {"x": _normal(gen, (b, t, h + 2 * n, hd), 1.0, dtype), "k": _normal(gen, (pages, c["page"], n, hd), 1.0, dtype),
             "v": _normal(gen, (pages, c["page"], n, hd), 1.0, dtype)}
    first = gen.integers(c["past"] // 2, c["past"] + 1, b).astype(np.int32)
    first[0] = c["past"]
    if b > 2:
        first[1] = 0  # a conversation that begins
    state["first"] = first
    data["table"] = gen.permutation(pages)[:b * each].reshape(b, each).astype(np.int32)
    data["drive"] = _normal(gen, state["x"].shape, 0.7, dtype)
    if c["slopes"]:
        data["slopes"] = _slopes(gen, h, dtype)
    if c["ragged"]:
        lengths = gen.integers(0, t + 1, b).astype(np.int32)
        lengths[0] = t
        data["lengths"] = lengths
    return state, data


def _rate(c, name):
    """Of a value read by a group of heads, and of a slope, whose gradient adds up every score."""
    if name == "slopes":
        return _RATE / (c["batch"] * c["length"] ** 2)
    return _RATE * c["keys"] / c["heads"]


def _max_norm(c):
    return 0.35 * math.sqrt(sum(math.prod(s) for s in _shapes(c).values()))


# ---- the framework's programs, as a user writes them ----------------------------------------------

def _own_attend(c, s, data):
    import rustautograd_amd as rg
    q, k, v = (s["x"], None, None) if c["joined"] else (s["q"], s["k"], s["v"])
    return rg.attention(q, k, v, heads=(c["heads"], c["keys"]) if c["joined"] else None, causal=c["causal"], cap=c["cap"] or None, slopes=s.get("slopes"),
                        documents=data.get("documents"), prefix=data.get("prefix"), lengths=data.get("lengths"))


def _own_step(c):
    import rustautograd_amd as rg
    from rustautograd_amd import optim

    def attend(s, data):
        def loss(s):
            off = _own_attend(c, s, data) - data["t"]
            return 0.5 * (off * off).sum()

        value, grads = rg.value_and_grad(loss)(s)
        return {k: s[k] - _rate(c, k) * grads[k] for k in s}, (value, grads)

    def cached(s, data):
        y, (k, v) = rg.paged_attention(s["x"], cache=(s["k"], s["v"]), table=data["table"], first=s["first"], lengths=data.get("lengths"),
                                       heads=(c["heads"], c["keys"]), cap=c["cap"] or None, slopes=data.get("slopes"))
        n = c["keys"]
        x = rg.tanh(0.5 * rg.concatenate([y, y[:, :, :n], y[:, :, c["heads"] - n:]], axis=2) + data["drive"])
        return {"x": x, "k": k, "v": v, "first": s["first"] + (data["lengths"] if c["ragged"] else c["length"])}

    def clip(s, data):
        grads, norm = optim.clip_gradients({k: s[k] - data[k] for k in s}, _max_norm(c))
        return {k: s[k] - _RATE * grads[k] for k in s}, norm

    return {"attend": attend, "cached": cached, "clip": clip}[c["kind"]]


def prepare(case, seed):
    """Host data, and for the framework's side the compiled program that a user keeps."""
    state, data = _inputs(case, seed)
    made = {"case": case, "state": state, "data": data}
    if own:
        import rustautograd_amd as rg
        made["state"], made["data"] = ({k: rg.tensor(v) for k, v in tree.items()} for tree in (state, data))
        made["program"] = rg.compile(_own_step(case), (made["state"], made["data"]), validate="basic")
    return made


def _joined_vectors(arrays):
    """Results as one dict of arrays, vectors joined into one."""
    out = {k: v for k, v in arrays.items() if v.ndim > 1 or k in ("loss", "norm", "first")}
    small = [arrays[k] for k in sorted(arrays) if k not in out]
    return {**out, "vectors": np.concatenate(small)} if small else out


def _own_pass(made):
    import rustautograd_amd as rg
    c = made["case"]
    r = rg.run(made["program"], made["state"], [made["data"]], steps=c["steps"])
    out = {k: v.numpy() for k, v in r.state.items()}
    if c["kind"] == "attend":
        out["loss"] = np.array(r.history["aux.0"], c["dtype"])
        out.update({"d" + k: v.numpy() for k, v in r.aux[1].items()})
    elif c["kind"] == "clip":
        out["norm"] = np.array(r.history["aux"], c["dtype"])
    return _joined_vectors(out)


# ---- the plain forms --------------------------------------------------------------------------------

def _up(tree, wide=False):
    out = {k: torch.from_numpy(np.ascontiguousarray(v)).to(_DEVICE) for k, v in tree.items()}
    return {k: v.double() if wide and v.is_floating_point() else v for k, v in out.items()}


def _down(tree):
    return {k: v.cpu().numpy() for k, v in tree.items()}


def _split(c, x):
    h, n = c["heads"], c["keys"]
    return x[:, :, :h], x[:, :, h:h + n], x[:, :, h + n:]


def _scores(c, q, k, slopes, apart):
    """Scaled, capped and biased scores [batch, heads, queries, keys] of q [batch, queries, heads,
    head] and k [batch, keys, heads, head]."""
    s = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(2, 3)) * (1.0 / math.sqrt(c["head"]))
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    if slopes is not None:
        s = s - slopes[:, None, None] * apart
    return s


def _weigh(s, seen, v):
    """The softmax over what is seen; a row that sees nothing is 0."""
    s = torch.where(seen, s, torch.full_like(s, -1e30))
    e = torch.exp(s - s.max(-1, keepdim=True).values.detach()) * seen
    z = e.sum(-1, keepdim=True)
    return ((e / torch.where(z > 0, z, torch.ones_like(z))) @ v.transpose(1, 2)).transpose(1, 2)


def _seen(c, data):
    """[batch, 1, queries, keys] truth: which keys a query sees."""
    t = c["length"]
    at = torch.arange(t, device=_DEVICE)
    seen = (at[None, :] <= at[:, None] if c["causal"] else torch.ones(t, t, dtype=torch.bool, device=_DEVICE))[None]
    if "prefix" in data:
        seen = seen | (at[None, None, :] < data["prefix"][:, None, None])
    if "documents" in data:
        ids = data["documents"]
        seen = seen & (ids[:, :, None] == ids[:, None, :]) & (ids[:, :, None] >= 0)
    if "lengths" in data:
        inside = at[None] < data["lengths"][:, None]
        seen = seen & inside[:, None, :] & inside[:, :, None]
    return seen.expand(c["batch"], t, t)[:, None]


def _plain_attend(c, s, data):
    q, k, v = _split(c, s["x"]) if c["joined"] else (s["q"], s["k"], s["v"])
    group = c["heads"] // c["keys"]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    at = torch.arange(c["length"], device=_DEVICE)
    apart = (at[:, None] - at[None, :]).abs().to(q.dtype)
    return _weigh(_scores(c, q, k, s.get("slopes"), apart), _seen(c, data), v)


def _descend(c, state, data, attend):
    at, losses, slopes = dict(state), [], ()
    for _ in range(c["steps"]):
        at = {k: v.detach().requires_grad_(True) for k, v in at.items()}
        value = 0.5 * ((attend(c, at, data) - data["t"]) ** 2).sum()
        slopes = torch.autograd.grad(value, list(at.values()))
        losses.append(value.detach())
        at = {k: (v - _rate(c, k) * g).detach() for (k, v), g in zip(at.items(), slopes)}
    return {**at, "loss": torch.stack(losses), **{"d" + k: g for k, g in zip(at, slopes)}}


def _follow(c, y, data):
    """The next tokens' queries, keys and values."""
    n = c["keys"]
    return torch.tanh(0.5 * torch.cat([y, y[:, :, :n], y[:, :, c["heads"] - n:]], 2) + data["drive"])


def _plain_cached(c, s, data):
    """One chunk: its keys and values go to their pages, then every query reads the pages."""
    b, t, page = c["batch"], c["length"], c["page"]
    q, k, v = _split(c, s["x"])
    table, new = data["table"].long(), torch.arange(t, device=_DEVICE)
    count = data["lengths"].long() if c["ragged"] else torch.full((b,), t, device=_DEVICE)
    place = s["first"].long()[:, None] + new
    row = torch.gather(table, 1, (place // page).clamp(max=table.shape[1] - 1)) * page + place % page
    inside = new[None] < count[:, None]
    flat = [pages.reshape(-1, c["keys"], c["head"]).clone() for pages in (s["k"], s["v"])]
    for pages, rows in zip(flat, (k, v)):
        pages[row[inside]] = rows[inside]
    keys, values = (pages.reshape(s["k"].shape)[table].reshape(b, -1, c["keys"], c["head"]) for pages in flat)
    group = c["heads"] // c["keys"]
    at = torch.arange(keys.shape[1], device=_DEVICE)
    apart = (place[:, :, None] - at).to(q.dtype)[:, None]
    seen = (at <= place[:, :, None]) & inside[:, :, None]
    y = _weigh(_scores(c, q, keys.repeat_interleave(group, 2), data.get("slopes"), apart), seen[:, None], values.repeat_interleave(group, 2))
    return {"x": _follow(c, y, data), "k": flat[0].reshape(s["k"].shape), "v": flat[1].reshape(s["v"].shape), "first": s["first"] + count.to(torch.int32)}


def _plain_clip(c, s, data):
    grads = {k: s[k] - data[k] for k in s}
    norm = torch.sqrt(sum((g.double() ** 2).sum() for g in grads.values()))
    factor = torch.clamp(_max_norm(c) / norm, max=1.0).to(grads["tok"].dtype)
    return {k: s[k] - _RATE * (grads[k] * factor) for k in s}, norm.to(factor.dtype)


def _repeat(c, state, data, cached, clip):
    if c["kind"] == "clip":
        norms = []
        for _ in range(c["steps"]):
            state, norm = clip(c, state, data)
            norms.append(norm)
        return {**state, "norm": torch.stack(norms)}
    for _ in range(c["steps"]):
        state = cached(c, state, data)
    return state


def _plain_pass(made):
    c, state, data = made["case"], _up(made["state"]), _up(made["data"])
    if c["kind"] == "attend":
        return _joined_vectors(_down(_descend(c, state, data, _plain_attend)))
    return _joined_vectors(_down(_repeat(c, state, data, _plain_cached, _plain_clip)))


def run(state):
    if own:
        return _own_pass(state)
    with torch.set_grad_enabled(state["case"]["kind"] == "attend"):
        return _plain_pass(state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    """A training step of attention reads its inputs twice (forward, backward) and the target, and
    writes the result, the gradients and the updated values; its products are two forward and five
    backward over the pairs that the causal order leaves. A token reads the keys and values before
    it and its own, and writes its own and its result. A clipped step reads parameters and targets
    for the norm and again for the update, which it writes."""
    c = case
    item, steps = 8 if c["dtype"] == "float64" else 4, c["steps"]
    if c["kind"] == "clip":
        n = float(sum(math.prod(s) for s in _shapes(c).values()))
        return {"bytes": steps * item * 5.0 * n, "flops": steps * 6.0 * n}
    b, t, h, n, hd = c["batch"], c["length"], c["heads"], c["keys"], c["head"]
    if c["kind"] == "attend":
        pairs = b * h * t * (t + 1) / 2 if c["causal"] else b * h * t * t
        if c["documents"]:
            pairs /= (c["documents"] + 1) / 2
        x, y = b * t * (h + 2 * n) * hd, b * t * h * hd
        return {"bytes": steps * item * (5.0 * x + 5.0 * y), "flops": steps * 14.0 * pairs * hd}
    seen = c["past"] * 0.75 if b > 1 else c["past"]
    return {"bytes": steps * item * b * (2.0 * n * hd * (seen + 2 * t) + 2.0 * t * h * hd), "flops": steps * 4.0 * b * h * t * (seen + t / 2) * hd}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _exact_row(c, q, k, v, slope, distance, seen):
    """One head of one sequence: the queries that see something, by the definition."""
    rows = seen.any(1)
    s = torch.einsum("id,jd->ij", q[rows], k) / math.sqrt(c["head"])
    if c["cap"]:
        s = c["cap"] - 2.0 * c["cap"] / (torch.exp(2.0 * s / c["cap"]) + 1.0)
    if slope is not None:
        s = s - slope * distance[rows]
    s = s.masked_fill(~seen[rows], -math.inf)
    y = torch.einsum("ij,jd->id", torch.exp(s - torch.logsumexp(s, 1, keepdim=True)), v)
    return torch.zeros_like(q).index_put((torch.nonzero(rows)[:, 0],), y)


def _exact_attend(c, s, data):
    q, k, v = _split(c, s["x"]) if c["joined"] else (s["q"], s["k"], s["v"])
    t, group = c["length"], c["heads"] // c["keys"]
    at = torch.arange(t, device=_DEVICE)
    distance, out = torch.abs(at[None] - at[:, None]).double(), []
    for b in range(c["batch"]):
        seen = torch.ones(t, t, dtype=torch.bool, device=_DEVICE)
        if c["causal"]:
            seen = seen.tril()
        if "prefix" in data:
            seen[:, :int(data["prefix"][b])] = True
        if "documents" in data:
            ids = data["documents"][b]
            seen = seen & (ids[None] == ids[:, None])
            seen[ids < 0] = False
        if "lengths" in data:
            seen[int(data["lengths"][b]):] = False
            seen[:, int(data["lengths"][b]):] = False
        slopes = s.get("slopes")
        out.append(torch.stack([_exact_row(c, q[b, :, h], k[b, :, h // group], v[b, :, h // group], None if slopes is None else slopes[h], distance, seen)
                                for h in range(c["heads"])], 1))
    return torch.stack(out)


def _exact_cached(c, s, data):
    """Sequence by sequence: its pages laid end to end, the new rows in their places."""
    q, new_k, new_v = _split(c, s["x"])
    pages_k, pages_v, first, out = s["k"].clone(), s["v"].clone(), s["first"].clone(), []
    for b in range(c["batch"]):
        count = int(data["lengths"][b]) if c["ragged"] else c["length"]
        begin = int(s["first"][b])
        for t in range(count):
            p, r = int(data["table"][b, (begin + t) // c["page"]]), (begin + t) % c["page"]
            pages_k[p, r], pages_v[p, r] = new_k[b, t], new_v[b, t]
        own_pages = data["table"][b, :-(-(begin + count) // c["page"])].long()
        k, v = (x[own_pages].flatten(0, 1)[:begin + count] for x in (pages_k, pages_v))
        query, key = torch.arange(begin, begin + count, device=_DEVICE), torch.arange(begin + count, device=_DEVICE)
        distance = (query[:, None] - key[None]).double()
        y = torch.zeros_like(q[b])
        for h in range(c["heads"] if count else 0):
            of = h // (c["heads"] // c["keys"])
            y[:count, h] = _exact_row(c, q[b, :count, h], k[:, of], v[:, of], data["slopes"][h] if c["slopes"] else None, distance, distance >= 0)
        out.append(y)
        first[b] += count
    return {"x": _follow(c, torch.stack(out), data), "k": pages_k, "v": pages_v, "first": first}


def _exact_clip(c, s, data):
    grads = {k: s[k] - data[k] for k in s}
    norm = torch.cat([g.flatten() for g in grads.values()]).square().sum().sqrt()
    if norm > _max_norm(c):
        grads = {k: g * (_max_norm(c) / norm) for k, g in grads.items()}
    return {k: s[k] - _RATE * grads[k] for k in s}, norm


def exact(case, seed):
    c = case
    state, data = (_up(tree, True) for tree in _inputs(c, seed))
    if c["kind"] == "attend":
        return _joined_vectors(_down(_descend(c, state, data, _exact_attend)))
    with torch.no_grad():
        return _joined_vectors(_down(_repeat(c, state, data, _exact_cached, _exact_clip)))
