"""The operators of a hybrid decoder's linear-attention layers and of its last
step whose speed this library is measured by: the short causal convolution
behind a layer's input product, linear attention with a decay and a state for
each head, and the choice of a token from the vocabulary's logits, each called
as a program calls it (one command, its encodes, finish).

With `own` false, `run` computes the same from elementary torch operations, in
32 bits, and in 64 where 32 lose what matters: sums of log decays, and weights
next to the borders of a sampled set. Both sides start from the same inputs.

Head counts and channels are those of such decoders (16 key and 48 value heads
of 128, whose queries, keys and values are 10240 channels) and smaller ones,
lengths go from one token to a whole prompt, vocabularies to 248320.
"""
from __future__ import annotations

import functools
import math
import struct

import numpy as np
import torch

own = False

EPS = 1e-6
FRESH = 1 << 31  # a slot word with this bit: the sequence starts from zeros
CHUNK = 64


# ---- the cases ----

def listed() -> list[dict]:
    return [
        # Decode of one token: the convolutions of four layers; latency counts.
        _conv("conv_token", channels=10240, width=4, batch=1, new=1, layers=4),
        # Prompts of three requests in one step, one of them continued.
        _conv("conv_prompts", channels=10240, width=4, batch=3, new=1367, fresh="some", ragged=True, layers=1),
        # Decode of one token: four layers in a command; latency counts.
        _linear("linear_token", k_heads=16, v_heads=48, dk=128, dv=128, batch=1, new=1, layers=4),
        # Decode of 32 sequences: their states are what has to move.
        _linear("linear_batch_32", k_heads=16, v_heads=48, dk=128, dv=128, batch=32, new=1, layers=1),
        # Verification of three drafted tokens, which leaves the states alone.
        _linear("linear_verify_3", k_heads=16, v_heads=48, dk=128, dv=128, batch=1, new=3, keep=False, layers=1),
        # A whole prompt at once.
        _linear("linear_prompt_4100", k_heads=16, v_heads=48, dk=128, dv=128, batch=1, new=4100, fresh="all", layers=1),
        # Chunks of several requests at once, ragged, some of them new.
        _linear("linear_ragged_7", k_heads=16, v_heads=32, dk=128, dv=128, batch=7, new=333, fresh="some",
                ragged=True, layers=1),
        # Plain linear attention, each head with a decay of its own that no token changes.
        _linear("linear_fixed_decay", k_heads=8, v_heads=8, dk=64, dv=128, batch=2, new=1011, delta=False, gates=False,
                qk_norm=False, out_norm=False, layers=1),
        # The token of one request: a few candidates kept.
        _sample("sample_token", rows=1, vocab=248320, k=20, p=0.95, min_p=0.0),
        # The same without a bound on their number.
        _sample("sample_nucleus", rows=1, vocab=248320, k=0, p=0.95, min_p=0.0),
        # A batch whose requests have settings of their own, a greedy one among them.
        _sample("sample_batch_48", rows=48, vocab=248320, k=40, p=0.9, min_p=0.02, mixed=True),
        # A small vocabulary.
        _sample("sample_small", rows=5, vocab=32001, k=0, p=1.0, min_p=0.05),
    ]


def _conv(name=None, *, channels, width, batch, new, layers, fresh="none", ragged=False, bias=False) -> dict:
    case = {"op": "conv", "channels": channels, "width": width, "batch": batch, "new": new, "fresh": fresh,
            "ragged": ragged, "bias": bias, "layers": layers}
    return {"name": name, **case} if name else case


def _linear(name=None, *, k_heads, v_heads, dk, dv, batch, new, layers, keep=True, fresh="none", ragged=False,
            delta=True, gates=True, qk_norm=True, out_norm=True) -> dict:
    case = {"op": "linear", "k_heads": k_heads, "v_heads": v_heads, "dk": dk, "dv": dv, "batch": batch, "new": new,
            "keep": keep, "fresh": fresh, "ragged": ragged, "delta": delta, "gates": gates, "qk_norm": qk_norm,
            "out_norm": out_norm, "layers": layers}
    return {"name": name, **case} if name else case


def _sample(name=None, *, rows, vocab, k, p, min_p, mixed=False) -> dict:
    case = {"op": "sample", "rows": rows, "vocab": vocab, "k": k, "p": p, "min_p": min_p, "mixed": mixed}
    return {"name": name, **case} if name else case


HEADS = [(16, 48, 128, 128), (16, 48, 128, 128), (16, 32, 128, 128), (4, 8, 64, 64), (8, 8, 64, 128), (2, 6, 96, 80),
         (1, 3, 256, 192), (5, 5, 40, 24)]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))))) if high > low else low))


def draw(rng) -> dict:
    """A case of the listed kinds, sizes over their whole ranges."""
    op = rng.choice(["conv", "linear", "linear", "linear", "sample", "sample"])
    if op == "sample":
        rows = _log(rng, 1, 48)
        return _sample(rows=rows, vocab=_log(rng, 1000, 248320), k=rng.choice([0, 0, 1, _log(rng, 2, 500)]),
                       p=rng.choice([1.0, round(rng.uniform(0.1, 0.999), 3)]),
                       min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 3)]), mixed=rows > 1 and rng.random() < 0.5)
    batch = _log(rng, 1, 48)
    fresh, ragged = rng.choice(["none", "some", "all"]), batch > 1 and rng.random() < 0.6
    if op == "conv":
        channels = _log(rng, 100, 10240)
        return _conv(channels=channels, width=rng.randint(2, 4), batch=batch,
                     new=rng.choice([1, rng.randint(2, 5), _log(rng, 2, max(2, 4100 // batch))]), fresh=fresh,
                     ragged=ragged, bias=rng.random() < 0.3, layers=1)
    k_heads, v_heads, dk, dv = rng.choice(HEADS)
    form = rng.choice(["token", "few", "chunk", "chunk"])
    most = max(6, 4100 // batch)
    new = 1 if form == "token" else rng.randint(2, 5) if form == "few" else _log(rng, 6, most)
    delta = rng.random() < 0.7
    return _linear(k_heads=k_heads, v_heads=v_heads, dk=dk, dv=dv, batch=batch, new=new, keep=rng.random() < 0.8,
                   fresh=fresh, ragged=ragged, delta=delta, gates=rng.random() < 0.7,
                   qk_norm=delta or rng.random() < 0.5, out_norm=rng.random() < 0.7, layers=1)


# ---- inputs, made from the seed alone ----

def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda")


def _uniform(g: torch.Generator, low: float, high: float, *shape: int) -> torch.Tensor:
    return low + (high - low) * torch.rand(shape, generator=g, device="cuda")


def _counts(case: dict) -> list[int]:
    """New tokens of every sequence."""
    draw_ = np.random.RandomState(case["batch"] * 7919 + case["new"])
    n = case["new"]
    return [int(draw_.randint(max(1, n // 3), n + 1)) if case["ragged"] else n for _ in range(case["batch"])]


def _slots(case: dict, seed: int) -> torch.Tensor:
    """int64 [batch]: places in a pool of some more, in no order; fresh ones marked."""
    order = np.random.RandomState((seed + 1) % (1 << 31)).permutation(case["batch"] + 3)[:case["batch"]]
    every = {"none": 0, "some": 2, "all": 1}[case["fresh"]]
    return torch.tensor([int(s) | (FRESH if every and i % every == 0 else 0) for i, s in enumerate(order)])


def _inputs(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # A broad floor, and some tokens that stand out of it.
        x = 2.5 * _normal(g, rows, vocab)
        x += 12 * (_uniform(g, 0, 1, rows, vocab) - (1 - 60 / vocab)).clamp(min=0) * (vocab / 60)
        t = {"logits": x, "uniform": torch.rand((rows,), generator=g, device="cuda")}
        row = torch.arange(rows, device="cuda")
        odd = (row % 3 == 1) if case["mixed"] else torch.zeros_like(row, dtype=torch.bool)
        t["temperature"] = torch.where(odd, 1.1, 0.7) * (row % 7 != 5 if case["mixed"] else 1)  # 0 is greedy
        t["top_k"] = torch.where(odd, 0, case["k"]).int()
        t["top_p"] = torch.where(odd, 0.95, case["p"]).float()
        t["min_p"] = torch.where(odd, 0.0, case["min_p"]).float()
        return t
    counts, layers = _counts(case), range(case["layers"])
    tokens, pool = sum(counts), case["batch"] + 3
    t = {"tokens": tokens, "longest": max(counts), "slots": _slots(case, seed),
         "starts": torch.tensor([0, *np.cumsum(counts)])}
    if case["op"] == "conv":
        c, w = case["channels"], case["width"]
        t["x"] = [_normal(g, tokens, c) for _ in layers]
        t["w"] = [_normal(g, c, w) / math.sqrt(w) for _ in layers]
        t["bias"] = [0.1 * _normal(g, c) for _ in layers]
        t["state"] = [_normal(g, pool, w - 1, c) for _ in layers]
        return t
    k_heads, v_heads, dk, dv = (case[n] for n in ("k_heads", "v_heads", "dk", "dv"))
    # Queries, keys and values as the convolution leaves them (SiLU of sums of
    # unit size), the other rows as products give them.
    mixed = 2 * k_heads * dk + v_heads * dv
    size = 1.0 if case["qk_norm"] else 1 / math.sqrt(dk)
    t["qkv"] = [torch.nn.functional.silu(_normal(g, tokens, mixed)) * size for _ in layers]
    t["z"] = [_normal(g, tokens, v_heads * dv) for _ in layers]
    t["b"] = [_normal(g, tokens, v_heads) for _ in layers]
    t["a"] = [_normal(g, tokens, v_heads) if case["gates"] else
              torch.log1p(-torch.exp2(-_uniform(g, 3, 10, 1, v_heads))) for _ in layers]
    t["a_log"] = [_uniform(g, 1, 16, v_heads).log() for _ in layers]
    # softplus of the step's bias lies between 0.001 and 0.1.
    t["dt_bias"] = [_uniform(g, math.log(0.001), math.log(0.1), v_heads).exp().expm1().log() for _ in layers]
    t["norm"] = [1 + 0.1 * _normal(g, dv) for _ in layers]
    t["state"] = [0.3 * _normal(g, pool, v_heads, dk, dv) for _ in layers]
    return t


# ---- the program ----

@functools.lru_cache(maxsize=None)
def _qmr():
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "qwen-mlx-runner_amd"))
    import qmr

    return qmr


@functools.lru_cache(maxsize=None)
def _gpu():
    return _qmr().Gpu("aligned")


def _word(v: float) -> int:
    return struct.unpack("<I", struct.pack("<f", v))[0]


class DeviceOutputs(dict):
    """Output buffers by name. They stay on the device; looking at one copies
    it to the host."""

    def __getitem__(self, name):
        buffer, shape, kind = super().__getitem__(name)
        return buffer.read(kind, math.prod(shape)).reshape(shape)


def prepare(case: dict, seed: int) -> dict:
    t = _inputs(case, seed)
    state = {"case": case, "t": {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in t.items()}}
    if own:
        state["calls"], state["out"] = _program(case, t)
    return state


def _program(case: dict, t: dict):
    """The dispatches of a pass, over buffers on the device, and its outputs."""
    gpu, q = _gpu(), _qmr()
    calls, out = [], {}

    def up(v, kind=torch.float32):
        v = v.cpu().to(kind).contiguous()
        return gpu.upload_bytes(v.numpy())

    def word(v):
        return gpu.upload_bytes(v.cpu().numpy().astype(np.uint32))

    def call(name, buffers, params, offsets=None):
        calls.append((name, buffers, params, q.dispatch_layout(name, params)[1], offsets))

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        tokens, probs = gpu.alloc(4 * rows), gpu.alloc_f32(rows)
        call("sample_logits", [up(t["logits"]), up(t["temperature"]), word(t["top_k"]), up(t["top_p"]), up(t["min_p"]),
                               up(t["uniform"]), tokens, probs], [rows, vocab, vocab])
        return calls, {"tokens": (tokens, (rows,), np.int32), "probs": (probs, (rows,), np.float32)}
    starts, slots, tokens, batch = word(t["starts"]), word(t["slots"]), t["tokens"], case["batch"]
    for i in range(case["layers"]):
        state, shape = up(t["state"][i]), tuple(t["state"][i].shape)
        if case["op"] == "conv":
            c = case["channels"]
            y = gpu.alloc_f32(tokens * c)
            call("conv_causal", [up(t["x"][i]), up(t["w"][i]), up(t["bias"][i]), starts, slots, state, y],
                 [batch, tokens, c, case["width"], c, c, 1, int(case["bias"]), shape[0], 1])
            out["y%d" % i] = (y, (tokens, c), np.float32)
        else:
            hk, hv, dk, dv = (case[n] for n in ("k_heads", "v_heads", "dk", "dv"))
            mixed, wide = 2 * hk * dk + hv * dv, hv * dv
            y, qkv = gpu.alloc_f32(tokens * wide), up(t["qkv"][i])
            call("attn_linear", [qkv, qkv, qkv, up(t["a"][i]), up(t["b"][i]), up(t["a_log"][i]), up(t["dt_bias"][i]),
                                 up(t["z"][i]), up(t["norm"][i]), starts, slots, state, y],
                 [batch, tokens, hk, hv, dk, dv, mixed, mixed, mixed, hv if case["gates"] else 0, hv, wide, wide,
                  t["longest"], int(case["gates"]), int(case["delta"]), _word(1 / math.sqrt(dk)),
                  _word(EPS) if case["qk_norm"] else 0, _word(EPS) if case["out_norm"] else 0, shape[0],
                  int(case["keep"])],
                 [0, 4 * hk * dk, 8 * hk * dk] + [0] * 10)
            out["o%d" % i] = (y, (tokens, hv, dv), np.float32)
        if case.get("keep", True):
            out["state%d" % i] = (state, shape, np.float32)
    return calls, out


def run(state: dict):
    if not own:
        form = {"conv": _plain_conv, "linear": _plain_linear, "sample": _plain_sample}[state["case"]["op"]]
        return form(state["case"], state["t"])
    command = _gpu().begin()
    for name, buffers, params, threads, offsets in state["calls"]:
        command.encode(name, buffers, params, threads, 64, offsets)
    command.finish()
    command.release()
    return DeviceOutputs(state["out"])


# ---- the plain forms: elementary operations ----

def _padded(t: dict):
    """(token [batch][longest], whether it is one, its place among all [tokens])."""
    starts = t["starts"]
    at = torch.arange(t["longest"], device=starts.device)
    token = starts[:-1, None] + at
    real = token < starts[1:, None]
    return token.clamp(max=t["tokens"] - 1), real, real.flatten().nonzero()[:, 0]


def _plain_conv(case: dict, t: dict) -> dict:
    w, count = case["width"], t["starts"][1:] - t["starts"][:-1]
    token, real, place = _padded(t)
    slot, fresh = t["slots"] % FRESH, t["slots"] >= FRESH
    tail = count[:, None] + torch.arange(w - 1, device=count.device)  # the last inputs, of state and tokens together

    def layer(i):
        x, state = t["x"][i], t["state"][i]
        old = state[slot].masked_fill(fresh[:, None, None], 0)
        rows = torch.cat([old, x[token] * real[..., None]], dim=1)
        y = (rows.unfold(1, w, 1) * t["w"][i]).sum(dim=-1).flatten(0, 1)[place]
        if case["bias"]:
            y = y + t["bias"][i]
        state[slot] = rows.gather(1, tail[..., None].expand(-1, -1, x.shape[1]))
        return {"y%d" % i: y * torch.sigmoid(y), "state%d" % i: state}

    return {k: v for i in range(case["layers"]) for k, v in layer(i).items()}


def _plain_linear(case: dict, t: dict) -> dict:
    return {k: v for i in range(case["layers"]) for k, v in _plain_linear_layer(case, t, i).items()}


def _chunks(x: torch.Tensor, size: int) -> torch.Tensor:
    """[batch][tokens][heads][..] as [batch][heads][chunk][size][..], zeros behind the last token."""
    pad = -x.shape[1] % size
    x = torch.cat([x, x.new_zeros(x.shape[0], pad, *x.shape[2:])], dim=1) if pad else x
    return x.unflatten(1, (-1, size)).movedim(3, 1)


def _inverse(a: torch.Tensor) -> torch.Tensor:
    """(I + a)^-1 of strictly lower triangles: a product of I + (-a)^(2^i)."""
    eye = torch.eye(a.shape[-1], device=a.device)
    result, power = eye - a, a @ a
    for _ in range(max(0, (a.shape[-1] - 1).bit_length() - 1)):
        result, power = result + result @ power, power @ power
    return result


def _plain_linear_layer(case: dict, t: dict, i: int) -> dict:
    hk, hv, dk, dv = (case[n] for n in ("k_heads", "v_heads", "dk", "dv"))
    token, real, place = _padded(t)
    size = min(CHUNK, t["longest"])
    mixed = t["qkv"][i][token] * real[..., None]
    q, k, v = mixed.split([hk * dk, hk * dk, hv * dv], dim=-1)
    q, k, v = q.unflatten(-1, (hk, dk)), k.unflatten(-1, (hk, dk)), v.unflatten(-1, (hv, dv))
    if case["qk_norm"]:
        q, k = (x * torch.rsqrt(x.square().sum(dim=-1, keepdim=True) + EPS) for x in (q, k))
    q, k = (_chunks(x.repeat_interleave(hv // hk, dim=2), size) for x in (q / math.sqrt(dk), k))
    v = _chunks(v, size)
    a = t["a"][i].expand(t["tokens"], hv)
    g = -t["a_log"][i].exp() * torch.nn.functional.softplus(a + t["dt_bias"][i]) if case["gates"] else a
    g = _chunks((g[token] * real[..., None]).double(), size).cumsum(dim=-1)  # [batch][heads][chunk][size]
    lower = torch.ones(size, size, device=g.device).tril()
    decay = (g[..., :, None] - g[..., None, :]).masked_fill(lower == 0, -math.inf).exp().float()
    left, last = g.exp().float()[..., None], (g[..., -1:] - g).exp().float()[..., None]
    whole = g[..., -1].exp().float()[..., None, None]
    u = v
    if case["delta"]:
        beta = _chunks(torch.sigmoid(t["b"][i][token]) * real[..., None], size)[..., None]
        solve = _inverse((beta * (k @ k.transpose(-1, -2)) * decay).tril(-1))
        u, w = solve @ (beta * v), solve @ (beta * left * k)
    inside, q, k = (q @ k.transpose(-1, -2)) * decay, q * left, k * last
    slot = t["slots"] % FRESH
    s = t["state"][i][slot].masked_fill((t["slots"] >= FRESH)[:, None, None, None], 0)
    out = torch.empty_like(v)
    for n in range(v.shape[2]):
        new = u[:, :, n] - w[:, :, n] @ s if case["delta"] else u[:, :, n]
        out[:, :, n] = q[:, :, n] @ s + inside[:, :, n] @ new
        s = whole[:, :, n] * s + k[:, :, n].transpose(-1, -2) @ new
    out = out.movedim(1, 3).flatten(1, 2)[:, :t["longest"]].flatten(0, 1)[place]
    if case["out_norm"]:
        z = t["z"][i].view(-1, hv, dv)
        out = out * torch.rsqrt(out.square().mean(dim=-1, keepdim=True) + EPS) * t["norm"][i] * z * torch.sigmoid(z)
    if not case["keep"]:
        return {"o%d" % i: out}
    t["state"][i][slot] = s
    return {"o%d" % i: out, "state%d" % i: t["state"][i]}


def _plain_sample(case: dict, t: dict) -> dict:
    x = t["logits"]
    warm = t["temperature"][:, None] > 0
    order = x.sort(dim=-1, descending=True, stable=True)
    weight = ((order.values.double() - order.values[:, :1].double()) / t["temperature"][:, None].double()).exp()
    rank = torch.arange(x.shape[1], device=x.device)
    weight = torch.where(warm, weight, (rank == 0).double())
    k = t["top_k"][:, None]
    weight = weight * ((rank < k) | (k == 0))
    before = weight.cumsum(dim=-1) - weight
    p = t["top_p"][:, None].double()
    weight = weight * ((before < p * weight.sum(dim=-1, keepdim=True)) | (p >= 1)) * (weight >= t["min_p"][:, None])
    weight = torch.zeros_like(weight).scatter_(1, order.indices, weight)
    up_to = weight.cumsum(dim=-1)
    total = up_to[:, -1:]
    token = (up_to <= t["uniform"][:, None].double() * total).sum(dim=-1, keepdim=True)
    return {"tokens": token[:, 0].int(), "probs": (weight.gather(1, token) / total)[:, 0].float()}


# ---- what a pass cannot do without ----

def work(case: dict) -> dict:
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 28.0 * case["rows"], "flops": 4.0 * n}
    tokens, layers = sum(_counts(case)), case["layers"]
    states = sum((1 if s < FRESH else 0) + (1 if case.get("keep", True) else 0) for s in _slots(case, 0).tolist())
    if case["op"] == "conv":
        c, w = case["channels"], case["width"]
        return {"bytes": 4.0 * layers * c * (2 * tokens + w + states * (w - 1)), "flops": layers * 2.0 * tokens * c * (w + 2)}
    hk, hv, dk, dv = (case[n] for n in ("k_heads", "v_heads", "dk", "dv"))
    row = 2 * hk * dk + 2 * hv * dv + (hv * dv if case["out_norm"] else 0) + hv * (case["gates"] + case["delta"])
    return {"bytes": 4.0 * layers * (tokens * row + states * hv * dk * dv),
            "flops": layers * float(tokens) * hv * dk * dv * (7 if case["delta"] else 5)}


# ---- from the definition, in 64 bits ----

def exact(case: dict, seed: int):
    t = _inputs(case, seed)
    if case["op"] == "sample":
        return _sample64(t)
    form = _conv64 if case["op"] == "conv" else _linear64
    return {k: v for i in range(case["layers"]) for k, v in form(case, t, i).items()}


def _conv64(case: dict, t: dict, i: int) -> dict:
    x, w, state = t["x"][i].double(), t["w"][i].double(), t["state"][i].double()
    starts, y = t["starts"].tolist(), torch.zeros_like(x)
    for b, word in enumerate(t["slots"].tolist()):
        s = word % FRESH
        rows = torch.cat([state[s] * (word < FRESH), x[starts[b]:starts[b + 1]]])
        n = starts[b + 1] - starts[b]
        for j in range(case["width"]):
            y[starts[b]:starts[b + 1]] += rows[j:j + n] * w[:, j]
        state[s] = rows[n:]
    y += t["bias"][i].double() * case["bias"]
    return {"y%d" % i: y / (1 + torch.exp(-y)), "state%d" % i: state}


def _linear64(case: dict, t: dict, i: int) -> dict:
    """Token after token, all sequences that have one together."""
    hk, hv, dk, dv = (case[n] for n in ("k_heads", "v_heads", "dk", "dv"))
    rows = t["qkv"][i].double()
    q, k = rows[:, :hk * dk].view(-1, hk, dk), rows[:, hk * dk:2 * hk * dk].view(-1, hk, dk)
    v = rows[:, 2 * hk * dk:].view(-1, hv, dv)
    if case["qk_norm"]:
        q, k = q / (q.pow(2).sum(-1, keepdim=True) + EPS).sqrt(), k / (k.pow(2).sum(-1, keepdim=True) + EPS).sqrt()
    head = torch.arange(hv, device=rows.device) // (hv // hk)
    a = t["a"][i].double()
    if case["gates"]:
        a = -torch.exp(t["a_log"][i].double()) * torch.log1p(torch.exp(a + t["dt_bias"][i].double()))
    keep = torch.exp(a).expand(len(rows), hv)
    beta = 1 / (1 + torch.exp(-t["b"][i].double()))
    starts, slots = t["starts"].to(rows.device), t["slots"].to(rows.device)
    state = t["state"][i].double()
    s = state[slots % FRESH] * (slots < FRESH)[:, None, None, None]
    out = torch.zeros(len(rows), hv, dv, dtype=torch.float64, device=rows.device)
    counts = (starts[1:] - starts[:-1]).tolist()
    first = starts.tolist()
    for n in range(max(counts)):
        live = [b for b, c in enumerate(counts) if c > n]
        at = torch.tensor([first[b] + n for b in live], device=rows.device)
        every = len(live) == len(counts)
        part = s if every else s[live]
        kt, vt = k[at][:, head], v[at]
        part = part * keep[at][..., None, None]
        if case["delta"]:
            vt = beta[at][..., None] * (vt - (part * kt[..., None]).sum(dim=-2))
        part = part + kt[..., None] * vt[..., None, :]
        out[at] = (part * q[at][:, head][..., None]).sum(dim=-2) / math.sqrt(dk)
        if every:
            s = part
        else:
            s[live] = part
    if case["out_norm"]:
        z = t["z"][i].double().view(-1, hv, dv)
        out = out / (out.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * t["norm"][i].double() * z / (1 + torch.exp(-z))
    if not case["keep"]:
        return {"o%d" % i: out}
    state[slots % FRESH] = s
    return {"o%d" % i: out, "state%d" % i: state}


def _sample64(t: dict) -> dict:
    """Row after row on the host."""
    x = t["logits"].cpu().numpy()
    tokens, probs = np.zeros(len(x), np.int32), np.zeros(len(x))
    options = [t[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "uniform")]
    for r, (row, temperature, k, p, min_p, u) in enumerate(zip(x, *options)):
        order = np.lexsort((np.arange(len(row)), -row))
        if temperature <= 0:
            tokens[r], probs[r] = order[0], 1.0
            continue
        w = np.exp((row[order].astype(np.float64) - float(row[order[0]])) / float(temperature))
        n = min(int(k), len(w)) if k else len(w)
        if p < 1:
            n = max(1, min(n, int(np.searchsorted(np.cumsum(w[:n]), float(p) * w[:n].sum(), side="left")) + 1))
        n = max(1, int(np.count_nonzero(w[:n] >= min_p)))
        kept = np.sort(order[:n])
        w = np.exp((row[kept].astype(np.float64) - float(row[order[0]])) / float(temperature))
        up_to = np.cumsum(w)
        at = min(int(np.searchsorted(up_to, float(u) * up_to[-1], side="right")), n - 1)
        tokens[r], probs[r] = kept[at], w[at] / up_to[-1]
    return {"tokens": tokens, "probs": probs}
