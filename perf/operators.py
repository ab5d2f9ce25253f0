"""The sequence operators of a hybrid decoder, as measurable cases.

Three operators carry a model's sense of time: a short depthwise causal convolution, the selective
state space scan it feeds, and the root-mean-square norm of each head's queries and keys (or of the
scan's input and output maps) with the rotation by position in the same pass. Each is trained, read
over prompts and stepped one token at a time; `nn.SelectiveSSM` runs the three together.

Tensors of this framework live in host memory between calls, so a case's pass is a whole call: its
inputs go to the device, the step loop (or the program) runs there, and what it returns comes back.
Training and generation take as many steps as put the device's work above the transfers; what comes
back is the state at the end and the last gradients, as a training or serving program keeps them.

Kinds of work (a case's `kind`):
- conv, scan, rotary: gradient descent on every input of one operator, as a layer inside a model
  meets it (inputs and parameters both have gradients), `steps` steps in one run.
- conv_tokens, scan_tokens, rotary_tokens: the form for single tokens, its state carried over
  `steps` tokens, each made from the last one's result.
- layer: gradient descent on the parameters and the input of one state space layer.
- layer_prompt: token ids in, the layer's output at every position and the state to go on from out;
  prompts of several lengths in one batch.
- layer_tokens: the same layer, one token a step for every sequence of a batch.
"""

import math

import numpy as np
import torch

own = False

_DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
_RATE = 0.05    # of a value read once; others take it divided by the number of terms in their gradient
_EPS, _BASE = 1e-6, 10000.0


def listed():
    return [
        # A convolution inside a small model being trained: 4 taps and SiLU, bias.
        {"name": "conv train 4x1024x512", "kind": "conv", "batch": 4, "length": 1024, "width": 512, "taps": 4, "ragged": False, "dtype": "float32",
         "steps": 200},
        # Prompts of several lengths padded to the longest, odd sizes, a state from before.
        {"name": "conv ragged 5x333x77", "kind": "conv", "batch": 5, "length": 333, "width": 77, "taps": 3, "ragged": True, "dtype": "float32",
         "steps": 64},
        # Sixteen sequences, one token a step.
        {"name": "conv tokens 16x2048", "kind": "conv_tokens", "batch": 16, "width": 2048, "taps": 4, "steps": 512},
        # The scan of a small model being trained, skip, gate and softplus in it.
        {"name": "scan train 2x2048x512", "kind": "scan", "batch": 2, "length": 2048, "width": 512, "states": 16, "groups": 1, "gated": True,
         "ragged": False, "dtype": "float32", "steps": 24},
        # Two groups of channels, 8 states, no gate, sequences of several lengths going on from a state.
        {"name": "scan ragged 3x777x200", "kind": "scan", "batch": 3, "length": 777, "width": 200, "states": 8, "groups": 2, "gated": False,
         "ragged": True, "dtype": "float32", "steps": 24},
        # Double precision, as used where gradients are checked.
        {"name": "scan f64 2x130x96", "kind": "scan", "batch": 2, "length": 130, "width": 96, "states": 16, "groups": 1, "gated": True,
         "ragged": False, "dtype": "float64", "steps": 24},
        # Sixteen sequences, one token a step.
        {"name": "scan tokens 16x2048", "kind": "scan_tokens", "batch": 16, "width": 2048, "states": 16, "groups": 1, "steps": 512},
        # Queries, keys and values of an attention layer being trained, 8 heads each.
        {"name": "rotary train 4x1024", "kind": "rotary", "batch": 4, "length": 1024, "queries": 8, "keys": 8, "values": 8, "head": 64,
         "turn": 64, "far": 0, "dtype": "float32", "steps": 100},
        # Grouped queries, half of an odd-sized head turned, positions far along.
        {"name": "rotary far 2x333", "kind": "rotary", "batch": 2, "length": 333, "queries": 6, "keys": 2, "values": 2, "head": 44,
         "turn": 22, "far": 1000000, "dtype": "float32", "steps": 64},
        # The whole layer of a small model being trained.
        {"name": "layer train 4x1024x256", "kind": "layer", "batch": 4, "length": 1024, "model": 256, "width": 512, "states": 16, "groups": 1,
         "taps": 4, "rank": 16, "steps": 24},
        # Reading two prompts.
        {"name": "layer prompt 2x2048x256", "kind": "layer_prompt", "batch": 2, "length": 2048, "model": 256, "width": 512, "states": 16,
         "groups": 1, "taps": 4, "rank": 16, "vocab": 96},
        # Going on from them, a token a step.
        {"name": "layer tokens 8x256", "kind": "layer_tokens", "batch": 8, "model": 256, "width": 512, "states": 16, "groups": 1, "taps": 4,
         "rank": 16, "steps": 128},
    ]


def _heads(c):
    return c["queries"] + c["keys"] + c["values"]


def _turned(c):
    """Heads of queries and of keys, which are normed and turned; the values' pass."""
    return [c["queries"], c["keys"]]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["conv", "conv", "conv_tokens", "scan", "scan", "scan", "scan_tokens", "rotary", "rotary", "rotary_tokens", "layer", "layer_prompt",
                       "layer_tokens"])
    dtype = rng.choice(["float32", "float32", "float32", "float64"])
    if kind == "conv":
        width, batch = _log_int(rng, 16, 1024), rng.randint(1, 6)
        most = max(8, 2 ** 20 // (width * batch))
        return {"kind": kind, "batch": batch, "length": _log_int(rng, 1, min(2048, most)), "width": width, "taps": rng.randint(2, 8),
                "ragged": rng.random() < 0.5, "dtype": dtype, "steps": rng.randint(24, 64)}
    if kind == "conv_tokens":
        return {"kind": kind, "batch": rng.randint(1, 16), "width": _log_int(rng, 32, 2048), "taps": rng.randint(2, 8), "steps": rng.randint(64, 256)}
    if kind in ("scan", "scan_tokens"):
        groups, states = rng.choice([1, 1, 2, 4]), rng.choice([1, 4, 8, 13, 16, 16, 16, 24, 32, 64])
        width = groups * _log_int(rng, 8, 512 // groups)
        if kind == "scan_tokens":
            return {"kind": kind, "batch": rng.randint(1, 16), "width": width, "states": states, "groups": groups, "steps": rng.randint(64, 256)}
        batch = rng.randint(1, 4)
        most = (2 ** 22 if dtype == "float64" else 2 ** 24) // (width * states * batch)
        return {"kind": kind, "batch": batch, "length": _log_int(rng, 1, max(16, min(2048, most))), "width": width, "states": states, "groups": groups,
                "gated": rng.random() < 0.6, "ragged": rng.random() < 0.4, "dtype": dtype, "steps": rng.randint(8, 24)}
    if kind in ("rotary", "rotary_tokens"):
        keys, head = rng.randint(1, 8), 2 * _log_int(rng, 4, 64)
        case = {"kind": kind, "batch": rng.randint(1, 4), "queries": keys * rng.choice([1, 2, 4]), "keys": keys, "values": rng.choice([0, keys]), "head": head,
                "turn": rng.choice([head, head, 2 * rng.randint(1, head // 2)]), "far": rng.choice([0, 0, rng.randint(1000, 2000000)])}
        if kind == "rotary_tokens":
            return {**case, "steps": rng.randint(64, 256)}
        most = max(8, 2 ** 21 // (case["batch"] * _heads(case) * head))
        return {**case, "length": _log_int(rng, 1, min(1024, most)), "dtype": dtype, "steps": rng.randint(24, 64)}
    groups, states = rng.choice([1, 2]), rng.choice([8, 16, 16, 32])
    model = 8 * rng.randint(4, 32)
    case = {"kind": kind, "batch": rng.randint(1, 4), "model": model, "width": groups * rng.randint(model // groups, 2 * model // groups), "states": states,
            "groups": groups, "taps": rng.randint(2, 4), "rank": rng.randint(4, 24)}
    if kind == "layer_tokens":
        return {**case, "steps": rng.randint(32, 128)}
    case["length"] = _log_int(rng, 30, min(1024, 2 ** 22 // (case["width"] * states) * 4 // case["batch"]))
    if kind == "layer_prompt":
        return {**case, "vocab": rng.randint(65, 130)}
    return {**case, "steps": rng.randint(8, 24)}


# ---- inputs -------------------------------------------------------------------------------------

def _normal(gen, shape, std, dtype=np.float32):
    return (gen.standard_normal(shape, dtype=np.float32) * np.float32(std)).astype(dtype)


def _lengths(gen, batch, length):
    """Lengths of a padded batch: one sequence fills it, one has a single token."""
    n = gen.integers(1, length + 1, batch).astype(np.int32)
    n[0] = length
    if batch > 1:
        n[-1] = 1
    return n


def _conv_weights(gen, taps, width, dtype=np.float32):
    return {"w": _normal(gen, (taps, width), 0.8 / math.sqrt(taps), dtype), "b": _normal(gen, (width,), 0.1, dtype)}


def _raw_steps(gen, shape, dtype=np.float32):
    """Step sizes before the softplus: steps from about 0.001 to 0.5."""
    size = np.exp(gen.uniform(math.log(0.001), math.log(0.5), shape))
    return np.log(np.expm1(size)).astype(dtype)


def _decays(gen, width, states, dtype=np.float32):
    """Decay rates -1, -2, ..., as such layers start from, moved a little by training."""
    return (-np.arange(1, states + 1, dtype=np.float64) * np.exp(0.1 * gen.standard_normal((width, states)))).astype(dtype)


def _scan_inputs(gen, c, length, dtype):
    b, d, n, g = c["batch"], c["width"], c["states"], c["groups"]
    x = {"x": _normal(gen, (b, length, d), 1.0, dtype), "dt": _raw_steps(gen, (b, length, d), dtype), "a": _decays(gen, d, n, dtype),
         "b": _normal(gen, (b, length, g, n), 1.0, dtype), "c": _normal(gen, (b, length, g, n), 1.0 / math.sqrt(n), dtype),
         "d": 1.0 + _normal(gen, (d,), 0.1, dtype), "h": _normal(gen, (b, d, n), 0.3, dtype)}
    if c.get("gated", True):
        x["z"] = _normal(gen, (b, length, d), 1.0, dtype)
    return x


def _layer_weights(gen, c):
    m, d, n, g, r = c["model"], c["width"], c["states"], c["groups"], c["rank"]
    return {"in": {"w": _normal(gen, (m, d), 1.0 / math.sqrt(m))}, "gate": {"w": _normal(gen, (m, d), 1.0 / math.sqrt(m))},
            "conv": _conv_weights(gen, c["taps"], d), "proj": {"w": _normal(gen, (d, r + 2 * g * n), 1.0 / math.sqrt(d))},
            "dt": {"w": _normal(gen, (r, d), 0.3 / math.sqrt(r)), "b": _raw_steps(gen, (d,))},
            "a_log": np.log(-_decays(gen, d, n)), "d": 1.0 + _normal(gen, (d,), 0.1), "gain": 1.0 + _normal(gen, (2, n), 0.1),
            "out": {"w": _normal(gen, (d, m), 1.0 / math.sqrt(d))}}


def _layer_state(gen, c):
    b, d = c["batch"], c["width"]
    return {"conv": _normal(gen, (b, c["taps"] - 1, d), 0.5), "scan": _normal(gen, (b, d, c["states"]), 0.3),
            "pos": gen.integers(0, 500, b).astype(np.int32)}


def _inputs(c, seed):
    """(state, data) of a case as trees of numpy arrays, from the seed alone. What is trained or
    carried from token to token is the state."""
    gen, kind, b = np.random.default_rng(seed), c["kind"], c["batch"]
    dtype = np.dtype(c.get("dtype", "float32"))
    if kind == "conv":
        shape = (b, c["length"], c["width"])
        state = {"x": _normal(gen, shape, 1.0, dtype), **_conv_weights(gen, c["taps"], c["width"], dtype),
                 "s": _normal(gen, (b, c["taps"] - 1, c["width"]), 1.0, dtype)}
        data = {"t": _normal(gen, shape, 0.5, dtype)}
    elif kind == "conv_tokens":
        state = {"x": _normal(gen, (b, 1, c["width"]), 1.0), "s": _normal(gen, (b, c["taps"] - 1, c["width"]), 1.0)}
        data = {**_conv_weights(gen, c["taps"], c["width"]), "drive": _normal(gen, (b, 1, c["width"]), 0.5)}
    elif kind == "scan":
        state = _scan_inputs(gen, c, c["length"], dtype)
        data = {"t": _normal(gen, state["x"].shape, 0.5, dtype)}
    elif kind == "scan_tokens":
        data = _scan_inputs(gen, c, 1, dtype)
        state = {"x": data.pop("x"), "h": data.pop("h")}
        data["drive"] = _normal(gen, state["x"].shape, 0.5)
    elif kind in ("rotary", "rotary_tokens"):
        length, heads = c.get("length", 1), _heads(c)
        state = {"x": _normal(gen, (b, length, heads, c["head"]), 1.0, dtype)}
        gain = 1.0 + _normal(gen, (2, c["head"]), 0.1, dtype)
        first = gen.integers(0, c["far"] + 1, (b, 1))
        position = (first + np.arange(length)).astype(np.int32)
        if kind == "rotary":
            state["gain"] = gain
            data = {"t": _normal(gen, state["x"].shape, 0.5, dtype), "pos": position}
        else:
            state["pos"] = position
            data = {"gain": gain, "drive": _normal(gen, state["x"].shape, 0.5)}
    elif kind == "layer":
        shape = (b, c["length"], c["model"])
        state, data = {"layer": _layer_weights(gen, c), "x": _normal(gen, shape, 1.0)}, {"t": _normal(gen, shape, 0.5)}
    elif kind == "layer_prompt":
        state = {"layer": _layer_weights(gen, c), "table": _normal(gen, (c["vocab"], c["model"]), 1.0)}
        data = {"ids": gen.integers(0, c["vocab"], (b, c["length"]), dtype=np.int32), "n": _lengths(gen, b, c["length"])}
    else:
        state = {"x": _normal(gen, (b, 1, c["model"]), 1.0), **_layer_state(gen, c)}
        data = {"layer": _layer_weights(gen, c), "drive": _normal(gen, (b, 1, c["model"]), 0.5)}
    if c.get("ragged"):
        data["n"] = _lengths(gen, b, c["length"])
        data["t"] *= np.arange(c["length"])[None, :, None] < data["n"][:, None, None]
    return state, data


def _map(f, tree):
    return {k: _map(f, v) for k, v in tree.items()} if isinstance(tree, dict) else f(tree)


def _leaves(tree, path=""):
    """(path, leaf) in a fixed order."""
    if isinstance(tree, dict):
        return [x for k in sorted(tree) for x in _leaves(tree[k], f"{path}.{k}")]
    return [(path.lstrip("."), tree)]


def _rebuild(tree, leaves, path=""):
    if isinstance(tree, dict):
        return {k: _rebuild(v, leaves, f"{path}.{k}") for k, v in tree.items()}
    return leaves[path.lstrip(".")]


def _trained(kind):
    return kind in ("conv", "scan", "rotary", "layer")


def _rate(c, path):
    kind, positions = c["kind"], c["batch"] * c["length"]
    if kind == "scan" and path in ("b", "c"):
        return _RATE * c["groups"] / c["width"]
    if path in ("x", "s", "h", "dt", "z"):
        return _RATE
    return _RATE / (positions * (_heads(c) if kind == "rotary" else 1))


def _output(tree):
    """A result as one dict of arrays, vectors and small tables joined."""
    out, small = {}, []
    for path, leaf in _leaves(tree):
        if path.startswith(("state", "grad")) and "loss" not in path and leaf.ndim < 2:
            small.append(leaf.reshape(-1))
        else:
            out[path] = leaf
    if small:
        out["vectors"] = np.concatenate(small)
    return out


# ---- the framework's programs, as a user writes them ----------------------------------------------

def _ssm(c):
    from rustautograd_amd import nn
    return nn.SelectiveSSM(c["model"], width=c["width"], states=c["states"], taps=c["taps"], dt_rank=c["rank"], groups=c["groups"], rotary=True)


def _own_result(c, s, data):
    """What a training case's operator makes of the state `s` it trains."""
    import rustautograd_amd as rg
    kind, n = c["kind"], data.get("n")
    if kind == "conv":
        return rg.causal_conv(s["x"], s["w"], s["b"], state=s["s"], lengths=n, activation="silu")[0]
    if kind == "scan":
        return rg.selective_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], d=s["d"], z=s.get("z"), state=s["h"], lengths=n, softplus=True)[0]
    if kind == "rotary":
        return rg.rotary_norm(s["x"], s["gain"], positions=data["pos"], sections=_turned(c), rotary_dims=c["turn"], base=_BASE, eps=_EPS)
    return _ssm(c)(s["layer"], s["x"])


def _own_training(c):
    import rustautograd_amd as rg

    def loss(s, data):
        off = _own_result(c, s, data) - data["t"]
        return 0.5 * (off * off).sum()

    def step(s, data):
        value, grads = rg.value_and_grad(loss)(s, data)
        at, slope = dict(_leaves(s)), dict(_leaves(grads))
        return _rebuild(s, {p: at[p] - _rate(c, p) * slope[p] for p in at}), (value, grads)

    return step


def _own_token(c):
    import rustautograd_amd as rg

    def step(s, data):
        if c["kind"] == "conv_tokens":
            y, carried = rg.causal_conv(s["x"], data["w"], data["b"], state=s["s"], activation="silu")
            return {"x": rg.tanh(0.5 * y + data["drive"]), "s": carried}
        if c["kind"] == "scan_tokens":
            y, carried = rg.selective_scan(s["x"], data["dt"], data["a"], data["b"], data["c"], d=data["d"], z=data["z"], state=s["h"], softplus=True)
            return {"x": rg.tanh(0.5 * y + data["drive"]), "h": carried}
        if c["kind"] == "rotary_tokens":
            y = rg.rotary_norm(s["x"], data["gain"], positions=s["pos"], sections=_turned(c), rotary_dims=c["turn"], base=_BASE, eps=_EPS)
            return {"x": 0.5 * y + data["drive"], "pos": s["pos"] + 1}
        y, carried = _ssm(c).extend(data["layer"], s["x"], {k: s[k] for k in ("conv", "scan", "pos")})
        return {"x": rg.tanh(0.2 * y + data["drive"]), **carried}

    return step


def _own_prompt(c, weights):
    import rustautograd_amd as rg

    def read(ids, lengths):
        return _ssm(c).extend(weights["layer"], rg.take(weights["table"], ids, 0), lengths=lengths)

    return read


def prepare(case, seed):
    """Host data, and for the framework's side the compiled program that a user keeps."""
    state, data = _inputs(case, seed)
    made = {"case": case, "state": state, "data": data}
    if own:
        import rustautograd_amd as rg
        made["state"], made["data"] = _map(rg.tensor, state), _map(rg.tensor, data)
        if case["kind"] == "layer_prompt":
            request = (made["data"]["ids"], made["data"]["n"])
            made["program"] = rg.compile(_own_prompt(case, made["state"]), request, validate="basic")
        else:
            step = _own_training(case) if _trained(case["kind"]) else _own_token(case)
            made["program"] = rg.compile(step, (made["state"], made["data"]), validate="basic")
    elif case["kind"] == "layer_prompt":
        made["weights"] = _map(_up, state)  # a serving program keeps them on the device
    return made


def _own_pass(made):
    import rustautograd_amd as rg
    c, fetch = made["case"], lambda tree: _map(lambda t: t.numpy(), tree)
    if c["kind"] == "layer_prompt":
        y, carried = made["program"](made["data"]["ids"], made["data"]["n"])
        return {"y": y.numpy(), **fetch(carried)}
    r = rg.run(made["program"], made["state"], [made["data"]], steps=c["steps"])
    if _trained(c["kind"]):
        return {"loss": np.array(r.history["aux.0"], c.get("dtype", "float32")), **_output({"state": fetch(r.state), "grad": fetch(r.aux[1])})}
    return _output(fetch(r.state))


# ---- the plain forms --------------------------------------------------------------------------------

def _up(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(_DEVICE)


def _inside(n, length):
    """[batch, length] truth: which positions belong to their sequence."""
    return torch.arange(length, device=_DEVICE)[None] < n[:, None]


def _plain_conv(x, w, b, s, n):
    taps, length = w.shape[0], x.shape[1]
    past = torch.cat([s, x], 1)
    y = b + sum(w[k] * past[:, k:k + length] for k in range(taps))
    y = y / (1 + torch.exp(-y))
    if n is None:
        return y, past[:, length:]
    at = n.long()[:, None] + torch.arange(taps - 1, device=_DEVICE)
    kept = torch.gather(past, 1, at[:, :, None].expand(-1, -1, x.shape[2]))
    return torch.where(_inside(n, length)[:, :, None], y, torch.zeros_like(y)), kept


def _plain_softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _plain_recurrence(decay, term):
    """h[t] = decay[t] h[t - 1] + term[t] along axis 1, by doubling."""
    span = 1
    while span < term.shape[1]:
        term = torch.cat([term[:, :span], term[:, span:] + decay[:, span:] * term[:, :-span]], 1)
        decay = torch.cat([decay[:, :span], decay[:, span:] * decay[:, :-span]], 1)
        span *= 2
    return term


def _spread(v, width):
    """[batch, length, groups, states] to one row of states for every channel."""
    return v.repeat_interleave(width // v.shape[2], 2)


def _plain_scan(p, n):
    x, dt, width = p["x"], _plain_softplus(p["dt"]), p["x"].shape[2]
    if n is not None:
        dt = torch.where(_inside(n, x.shape[1])[:, :, None], dt, torch.zeros_like(dt))
    decay = torch.exp(dt[..., None] * p["a"])
    term = (dt * x)[..., None] * _spread(p["b"], width)
    term = torch.cat([term[:, :1] + decay[:, :1] * p["h"][:, None], term[:, 1:]], 1)
    h = _plain_recurrence(decay, term)
    y = (h * _spread(p["c"], width)).sum(-1) + p["d"] * x
    if "z" in p:
        y = y * p["z"] / (1 + torch.exp(-p["z"]))
    if n is not None:
        y = torch.where(_inside(n, x.shape[1])[:, :, None], y, torch.zeros_like(y))
    return y, h[:, -1]


def _plain_rotary(x, gain, pos, sections, turn):
    """The angles of far positions need more than 32 bits."""
    half, used = turn // 2, sum(sections)
    inverse = _BASE ** (-torch.arange(half, device=_DEVICE, dtype=torch.float64) * 2 / turn)
    angle = pos[..., None, None].double() * inverse
    cos, sin = torch.cos(angle).to(x.dtype), torch.sin(angle).to(x.dtype)
    rows = gain.repeat_interleave(torch.tensor(sections, device=_DEVICE), 0)
    v = x[:, :, :used]
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + _EPS) * rows
    first, second = v[..., :half], v[..., half:turn]
    turned = torch.cat([first * cos - second * sin, second * cos + first * sin, v[..., turn:]], -1)
    return torch.cat([turned, x[:, :, used:]], 2)


def _plain_layer(c, p, x, s, n):
    """(output, carried state) of the state space layer on [batch, length, model]."""
    b, length, width, groups, states = x.shape[0], x.shape[1], c["width"], c["groups"], c["states"]
    gate = x @ p["gate"]["w"]
    u, kept = _plain_conv(x @ p["in"]["w"], p["conv"]["w"], p["conv"]["b"], s["conv"], n)
    maps = u @ p["proj"]["w"]
    dt = maps[..., :c["rank"]] @ p["dt"]["w"] + p["dt"]["b"]
    pos = s["pos"][:, None] + torch.arange(length, device=_DEVICE)
    maps = _plain_rotary(maps[..., c["rank"]:].reshape(b, length, 2 * groups, states), p["gain"], pos, [groups, groups], states)
    y, h = _plain_scan({"x": u, "dt": dt, "a": -torch.exp(p["a_log"]), "b": maps[:, :, :groups], "c": maps[:, :, groups:], "d": p["d"], "z": gate,
                        "h": s["scan"]}, n)
    return y @ p["out"]["w"], {"conv": kept, "scan": h, "pos": s["pos"] + (length if n is None else n)}


def _fresh(c, dtype=torch.float32):
    b, d = c["batch"], c["width"]
    return {"conv": torch.zeros(b, c["taps"] - 1, d, dtype=dtype, device=_DEVICE), "scan": torch.zeros(b, d, c["states"], dtype=dtype, device=_DEVICE),
            "pos": torch.zeros(b, dtype=torch.int32, device=_DEVICE)}


def _plain_result(c, s, data):
    kind, n = c["kind"], data.get("n")
    if kind == "conv":
        return _plain_conv(s["x"], s["w"], s["b"], s["s"], n)[0]
    if kind == "scan":
        return _plain_scan(s, n)[0]
    if kind == "rotary":
        return _plain_rotary(s["x"], s["gain"], data["pos"], _turned(c), c["turn"])
    return _plain_layer(c, s["layer"], s["x"], _fresh(c), n)[0]


def _descend(c, state, data, result):
    """The training loop: (updated state, loss of each step, last gradients)."""
    at, losses, slopes = dict(_leaves(state)), [], ()
    for _ in range(c["steps"]):
        at = {p: v.detach().requires_grad_(True) for p, v in at.items()}
        value = 0.5 * ((result(c, _rebuild(state, at), data) - data["t"]) ** 2).sum()
        slopes = torch.autograd.grad(value, list(at.values()))
        losses.append(value.detach())
        at = {p: (v - _rate(c, p) * g).detach() for (p, v), g in zip(at.items(), slopes)}
    return _rebuild(state, at), torch.stack(losses), _rebuild(state, dict(zip(at, slopes)))


def _plain_token(c, s, data):
    if c["kind"] == "conv_tokens":
        y, carried = _plain_conv(s["x"], data["w"], data["b"], s["s"], None)
        return {"x": torch.tanh(0.5 * y + data["drive"]), "s": carried}
    if c["kind"] == "scan_tokens":
        y, carried = _plain_scan({**data, **s}, None)
        return {"x": torch.tanh(0.5 * y + data["drive"]), "h": carried}
    if c["kind"] == "rotary_tokens":
        return {"x": 0.5 * _plain_rotary(s["x"], data["gain"], s["pos"], _turned(c), c["turn"]) + data["drive"], "pos": s["pos"] + 1}
    y, carried = _plain_layer(c, data["layer"], s["x"], s, None)
    return {"x": torch.tanh(0.2 * y + data["drive"]), **carried}


def _plain_pass(made):
    c, down = made["case"], lambda tree: _map(lambda t: t.cpu().numpy(), tree)
    data = _map(_up, made["data"])
    if c["kind"] == "layer_prompt":
        w = made["weights"]
        y, carried = _plain_layer(c, w["layer"], w["table"][data["ids"].long()], _fresh(c), data["n"])
        return {"y": y.cpu().numpy(), **down(carried)}
    state = _map(_up, made["state"])
    if _trained(c["kind"]):
        new, losses, slopes = _descend(c, state, data, _plain_result)
        return {"loss": losses.cpu().numpy(), **_output({"state": down(new), "grad": down(slopes)})}
    for _ in range(c["steps"]):
        state = _plain_token(c, state, data)
    return _output(down(state))


def run(state):
    if own:
        return _own_pass(state)
    with torch.set_grad_enabled(_trained(state["case"]["kind"])):
        return _plain_pass(state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def _scan_flops(positions, width, states):
    """Decay, update and output of every state: one exponential and five operations."""
    return 6.0 * positions * width * states


def _layer_flops(c, positions):
    d, m, maps = c["width"], c["model"], c["rank"] + 2 * c["groups"] * c["states"]
    return 2.0 * positions * (3 * m * d + d * maps + c["rank"] * d + c["taps"] * d) + _scan_flops(positions, d, c["states"])


def _layer_size(c):
    d, m, maps = c["width"], c["model"], c["rank"] + 2 * c["groups"] * c["states"]
    return 3 * m * d + d * maps + c["rank"] * d + (c["taps"] + c["states"] + 3) * d + 2 * c["states"]


def work(case):
    """A training step reads its inputs twice (forward, backward) and the target, and writes the
    result, the gradients and the updated values once; a token reads its weights, inputs and state
    and writes result and state."""
    c = case
    kind, b, steps, item = c["kind"], c["batch"], c.get("steps", 1), 8 if c.get("dtype") == "float64" else 4
    positions = b * c.get("length", 1)
    if kind == "conv":
        x = positions * c["width"]
        return {"bytes": steps * item * 7.0 * x, "flops": steps * x * (6.0 * c["taps"] + 12)}
    if kind == "conv_tokens":
        d = c["width"]
        return {"bytes": steps * 4.0 * d * (b * (2 * c["taps"] + 1) + c["taps"] + 1), "flops": steps * 2.0 * b * d * c["taps"]}
    if kind == "scan":
        d, n = c["width"], c["states"]
        size = positions * ((3 if c["gated"] else 2) * d + 2 * c["groups"] * n) + d * n + b * d * n
        return {"bytes": steps * item * (4.0 * size + 2 * positions * d), "flops": steps * 3.0 * _scan_flops(positions, d, n)}
    if kind == "scan_tokens":
        d, n = c["width"], c["states"]
        return {"bytes": steps * 4.0 * (b * d * (2 * n + 5) + d * n + 2 * b * c["groups"] * n), "flops": steps * _scan_flops(b, d, n)}
    if kind in ("rotary", "rotary_tokens"):
        x = positions * _heads(c) * c["head"]
        used = positions * sum(_turned(c)) * c["head"]
        if kind == "rotary":
            return {"bytes": steps * item * 6.0 * x, "flops": steps * 24.0 * used}
        return {"bytes": steps * 4.0 * 3 * x, "flops": steps * 8.0 * used}
    if kind == "layer":
        return {"bytes": steps * 4.0 * (4.0 * _layer_size(c) + 6.0 * positions * c["model"]), "flops": steps * 3.0 * _layer_flops(c, positions)}
    if kind == "layer_prompt":
        return {"bytes": 4.0 * (_layer_size(c) + positions * (1 + c["model"])), "flops": _layer_flops(c, positions)}
    return {"bytes": steps * 4.0 * (_layer_size(c) + 2 * b * c["width"] * (c["states"] + c["taps"] - 1)), "flops": steps * _layer_flops(c, b)}


# ---- the definitions in 64 bits -------------------------------------------------------------------

def _wide(x):
    x = _up(x)
    return x.double() if x.is_floating_point() else x


def _exact_conv(x, w, b, s, n):
    windows = torch.cat([s, x], 1).unfold(1, w.shape[0], 1)
    pre = torch.einsum("btdk,kd->btd", windows, w) + b
    y = torch.nn.functional.silu(pre)
    rows = []
    for i in range(x.shape[0]):
        last = x.shape[1] if n is None else int(n[i])
        rows.append(torch.cat([s[i], x[i, :last]], 0)[last:])
        if last < x.shape[1]:
            y = torch.cat([y[:i], torch.cat([y[i:i + 1, :last], torch.zeros_like(y[i:i + 1, last:])], 1), y[i + 1:]], 0)
    return y, torch.stack(rows)


_BLOCK = 16


def _exact_scan(p, n):
    """The recurrence solved block by block in closed form: h[t] is the start's state times the
    decay to t, and every term times the decay from its position to t."""
    x, width = p["x"], p["x"].shape[2]
    dt = torch.nn.functional.softplus(p["dt"], threshold=1000.0)
    if n is not None:
        dt = dt * _inside(n, x.shape[1])[:, :, None]
    h, out = p["h"], []
    per = width // p["b"].shape[2]
    for at in range(0, x.shape[1], _BLOCK):
        t, u = dt[:, at:at + _BLOCK], x[:, at:at + _BLOCK]
        b, c = (p[k][:, at:at + _BLOCK].repeat_interleave(per, 2) for k in ("b", "c"))
        span = torch.cumsum(t, 1)
        apart = span[:, :, None] - span[:, None]
        later = torch.ones(t.shape[1], t.shape[1], dtype=torch.bool, device=_DEVICE).tril()
        reach = torch.exp(apart[..., None] * p["a"]) * later[None, :, :, None, None]
        states = (reach * ((t * u)[..., None] * b)[:, None]).sum(2) + torch.exp(span[..., None] * p["a"]) * h[:, None]
        out.append((states * c).sum(-1))
        h = states[:, -1]
    y = torch.cat(out, 1) + p["d"] * x
    if "z" in p:
        y = y * torch.nn.functional.silu(p["z"])
    if n is not None:
        y = y * _inside(n, x.shape[1])[:, :, None]
    return y, h


def _exact_rotary(x, gain, pos, sections, turn):
    """The turn as a product of complex numbers."""
    half, at, parts = turn // 2, 0, []
    angle = pos.double()[..., None] * torch.exp(torch.arange(half, device=_DEVICE).double() * (-2.0 / turn * math.log(_BASE)))
    phase = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    for row, heads in enumerate(sections):
        v = x[:, :, at:at + heads]
        v = v * (v.square().mean(-1, keepdim=True) + _EPS).rsqrt() * gain[row]
        z = torch.complex(v[..., :half], v[..., half:turn]) * phase
        parts.append(torch.cat([z.real, z.imag, v[..., turn:]], -1))
        at += heads
    return torch.cat(parts + [x[:, :, at:]], 2)


def _exact_layer(c, p, x, s, n):
    u, kept = _exact_conv(x @ p["in"]["w"], p["conv"]["w"], p["conv"]["b"], s["conv"], n)
    low, maps = torch.split(u @ p["proj"]["w"], [c["rank"], 2 * c["groups"] * c["states"]], -1)
    pos = torch.arange(x.shape[1], device=_DEVICE) + s["pos"].long()[:, None]
    maps = _exact_rotary(maps.unflatten(-1, (2 * c["groups"], c["states"])), p["gain"], pos, [c["groups"], c["groups"]], c["states"])
    b, out = maps.split(c["groups"], 2)
    y, h = _exact_scan({"x": u, "dt": low @ p["dt"]["w"] + p["dt"]["b"], "a": -p["a_log"].exp(), "b": b, "c": out, "d": p["d"],
                        "z": x @ p["gate"]["w"], "h": s["scan"]}, n)
    return y @ p["out"]["w"], {"conv": kept, "scan": h, "pos": s["pos"] + (x.shape[1] if n is None else n)}


def _exact_result(c, s, data):
    kind, n = c["kind"], data.get("n")
    if kind == "conv":
        return _exact_conv(s["x"], s["w"], s["b"], s["s"], n)[0]
    if kind == "scan":
        return _exact_scan(s, n)[0]
    if kind == "rotary":
        return _exact_rotary(s["x"], s["gain"], data["pos"], _turned(c), c["turn"])
    return _exact_layer(c, s["layer"], s["x"], _fresh(c, torch.float64), n)[0]


def _exact_token(c, s, data):
    if c["kind"] == "conv_tokens":
        y, carried = _exact_conv(s["x"], data["w"], data["b"], s["s"], None)
        return {"x": (0.5 * y + data["drive"]).tanh(), "s": carried}
    if c["kind"] == "scan_tokens":
        y, carried = _exact_scan({**data, **s}, None)
        return {"x": (0.5 * y + data["drive"]).tanh(), "h": carried}
    if c["kind"] == "rotary_tokens":
        return {"x": 0.5 * _exact_rotary(s["x"], data["gain"], s["pos"], _turned(c), c["turn"]) + data["drive"], "pos": s["pos"] + 1}
    y, carried = _exact_layer(c, data["layer"], s["x"], s, None)
    return {"x": (0.2 * y + data["drive"]).tanh(), **carried}


def exact(case, seed):
    c, down = case, lambda tree: _map(lambda t: t.cpu().numpy(), tree)
    state, data = (_map(_wide, tree) for tree in _inputs(c, seed))
    if _trained(c["kind"]):
        new, losses, slopes = _descend(c, state, data, _exact_result)
        return {"loss": losses.cpu().numpy(), **_output({"state": down(new), "grad": down(slopes)})}
    with torch.no_grad():
        if c["kind"] == "layer_prompt":
            y, carried = _exact_layer(c, state["layer"], state["table"][data["ids"].long()], _fresh(c, torch.float64), data["n"])
            return {"y": y.cpu().numpy(), **down(carried)}
        for _ in range(c["steps"]):
            state = _exact_token(c, state, data)
    return _output(down(state))
