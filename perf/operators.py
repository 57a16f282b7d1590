"""The attention operators whose speed this library is measured by: rotary
positions with several axes, appending to a paged key-value cache, and
attention of new tokens over that cache, each called as a program calls it
(one command, its encodes, finish).

With `own` false, `run` computes the same from elementary torch operations in
32 bits. Both sides start from the same inputs, which a program has from its
host; the caches of the plain form are [page][head][slot][dim], those of the
library are stored as its operators take them.

Head counts and sizes are those of grouped-query decoders (24 query and 4
key-value heads of 256, 32 and 8 of 128, and smaller ones), lengths go from
one token to a whole prompt.
"""
from __future__ import annotations

import functools
import math
import struct

import numpy as np
import torch

own = False

EPS = 1e-6
HALF = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- the cases ----

def listed() -> list[dict]:
    return [
        # Decode of one token: the queries of four layers, positions of text
        # among images (three axes, dealt in turn); latency counts.
        _rope("rope_token", tokens=1, heads=24, dim=256, rotary=64, axes=3, dealt=True, layers=4),
        # A vision encoder's queries: a 64 x 68 grid of patches, two axes.
        _rope("rope_image", tokens=4352, heads=16, dim=72, rotary=72, axes=2, dealt=False, layers=1),
        # Decode of one token: normalise, rotate and append in four layers.
        _append("append_token", kind="bf16", heads=24, kv_heads=4, dim=256, rotary=64, axes=3, norm=True, batch=1,
                new=1, old=1000, page=64, layers=4),
        # Decode of a batch of 48 sequences, another head layout, no norm.
        _append("append_batch_48", kind="f16", heads=32, kv_heads=8, dim=128, rotary=128, axes=1, norm=False, batch=48,
                new=1, old=700, page=32, layers=1),
        # A prompt's chunk of 2011 tokens behind 1000 that are cached.
        _append("append_chunk_2011", kind="bf16", heads=24, kv_heads=4, dim=256, rotary=64, axes=3, norm=True, batch=1,
                new=2011, old=1000, page=64, layers=1),
        # Decode of one token with a short history, four layers in a command.
        _attend("attn_token_1001", kind="bf16", heads=24, kv_heads=4, dim=256, batch=1, new=1, old=1000, page=64,
                layers=4),
        # Decode of one token with a long history.
        _attend("attn_token_32k", kind="f16", heads=24, kv_heads=4, dim=256, batch=1, new=1, old=32767, page=128,
                layers=1),
        # Decode of a batch: histories of 1 to 8001 tokens.
        _attend("attn_batch_32", kind="bf16", heads=32, kv_heads=8, dim=128, batch=32, new=1, old=8000, page=64,
                ragged=True, layers=1),
        # Verification of three drafted tokens.
        _attend("attn_verify_3", kind="bf16", heads=24, kv_heads=4, dim=256, batch=1, new=3, old=12000, page=64,
                layers=1),
        # A prompt's chunk over a long history.
        _attend("attn_chunk_512_16k", kind="bf16", heads=24, kv_heads=4, dim=256, batch=1, new=512, old=16001,
                page=64, layers=1),
        # A whole prompt in one chunk.
        _attend("attn_prompt_4100", kind="f16", heads=32, kv_heads=8, dim=128, batch=1, new=4100, old=0, page=128,
                layers=1),
        # Chunks of several requests at once, ragged, with a sliding window.
        _attend("attn_ragged_window", kind="f16", heads=14, kv_heads=2, dim=64, batch=7, new=333, old=5000, page=32,
                window=1500, ragged=True, layers=1),
    ]


def _rope(name=None, *, tokens, heads, dim, rotary, axes, dealt, layers) -> dict:
    case = {"op": "rope", "tokens": tokens, "heads": heads, "dim": dim, "rotary": rotary, "axes": axes,
            "dealt": dealt, "adjacent": False, "layers": layers}
    return {"name": name, **case} if name else case


def _append(name=None, *, kind, heads, kv_heads, dim, rotary, axes, norm, batch, new, old, page, layers,
            ragged=False, adjacent=False) -> dict:
    case = {"op": "append", "kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "axes": axes, "dealt": axes > 1, "adjacent": adjacent, "norm": norm, "batch": batch, "new": new,
            "old": old, "page": page, "ragged": ragged, "layers": layers}
    return {"name": name, **case} if name else case


def _attend(name=None, *, kind, heads, kv_heads, dim, batch, new, old, page, layers, window=0, ragged=False) -> dict:
    case = {"op": "attend", "kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "batch": batch,
            "new": new, "old": old, "page": page, "window": window, "ragged": ragged, "layers": layers}
    return {"name": name, **case} if name else case


HEADS = [(24, 4, 256), (32, 8, 128), (20, 4, 256), (16, 2, 128), (14, 2, 64), (8, 8, 64), (10, 2, 80), (6, 1, 192)]


def _log(rng, low: int, high: int) -> int:
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v if v != 3072 else v + 1))


def draw(rng) -> dict:
    """A case of the listed kinds, sizes over their whole ranges."""
    op = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "attend"])
    heads, kv_heads, dim = rng.choice(HEADS)
    kind, page = rng.choice(["bf16", "f16"]), rng.choice([32, 64, 128, 256])
    if op == "rope":
        axes = rng.randint(1, 4)
        rotary = rng.choice([dim, dim // 2 // 2 * 2])
        tokens = _log(rng, 1, 4352)
        return _rope(tokens=tokens, heads=heads, dim=dim, rotary=rotary, axes=axes,
                     dealt=axes > 1 and rng.random() < 0.5, layers=rng.randint(1, 3) if tokens < 100 else 1)
    if op == "append":
        batch = _log(rng, 1, 64)
        return _append(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim // 2 // 2 * 2]),
                       axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.5, batch=batch,
                       new=_log(rng, 1, max(2, 2400 // batch)), old=_log(rng, 1, max(2, 4000 // batch)), page=page,
                       ragged=batch > 1 and rng.random() < 0.5, adjacent=rng.random() < 0.3, layers=1)
    form = rng.choice(["token", "token", "few", "chunk"])
    if form == "token":
        batch = _log(rng, 1, 64)
        new, old = 1, _log(rng, 10, max(100, min(40000, 120000 // batch)))
    elif form == "few":
        batch = _log(rng, 1, 8)
        new, old = rng.randint(2, 9), _log(rng, 10, 24000 // batch)
    else:
        batch = _log(rng, 1, 6)
        new, old = _log(rng, 16, 1200 // batch), _log(rng, 1, 6000 // batch)
    return _attend(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, batch=batch, new=new, old=old, page=page,
                   window=rng.choice([0, 0, 0, _log(rng, 20, 4000)]), ragged=batch > 1 and rng.random() < 0.6,
                   layers=1)


# ---- inputs, made from the seed alone ----

def _rng(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.randn(shape, generator=g, device="cuda")


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and cache length (new ones counted) of every sequence."""
    draw_ = np.random.RandomState(case["batch"] * 7919 + case["new"])
    new, old = [case["new"]] * case["batch"], [case["old"]] * case["batch"]
    if case["ragged"]:
        new = [int(draw_.randint(max(1, n // 3), n + 1)) for n in new]
        old = [int(draw_.randint(0, n + 1)) for n in old]
    return new, [n + o for n, o in zip(new, old)]


def _sections(rotary: int, axes: int) -> list[int]:
    """Pairs of each axis: near even, the first axis taking what is left."""
    pairs = rotary // 2
    rest = [pairs // axes] * (axes - 1)
    return [pairs - sum(rest), *rest] + [0] * (4 - axes)


def _axis_of(rotary: int, axes: int, dealt: bool) -> list[int]:
    """The axis whose position each pair of dimensions turns by."""
    n = _sections(rotary, axes)
    if not dealt:
        return [a for a in range(axes) for _ in range(n[a])]
    return [i % axes if i % axes and i < axes * n[i % axes] else 0 for i in range(rotary // 2)]


def _positions(case: dict, tokens: int, seed: int) -> torch.Tensor:
    """int32 [axes][tokens]: running positions on the first axis, places in a
    grid on the others."""
    t = torch.arange(tokens, dtype=torch.int32)
    base = 1000 + seed % 977
    return torch.stack([base + t, t // 68, t % 68, t // 7][:case["axes"]])


def _tables(case: dict, lengths: list[int], seed: int) -> tuple[torch.Tensor, int]:
    """(int32 [batch][columns], pages of the pool): pages in random order, as
    a pool that has been in use for a while gives them."""
    page = case["page"]
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 1
    order = np.random.RandomState((seed + 1) % (1 << 31)).permutation(pool)
    table = np.zeros((len(lengths), max(need)), np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table), pool


def _inputs(case: dict, seed: int) -> dict:
    g = _rng(seed)
    layers = range(case["layers"])
    if case["op"] == "rope":
        tokens = case["tokens"]
        return {"tokens": tokens, "positions": _positions(case, tokens, seed), "freqs": _freqs(case["rotary"]),
                "x": [_normal(g, tokens, case["heads"] * case["dim"]) for _ in layers]}
    new, lengths = _lengths(case)
    tokens = sum(new)
    table, pages = _tables(case, lengths, seed)
    t = {"tokens": tokens, "longest_new": max(new), "longest": max(lengths), "pages": pages, "table": table,
         "starts": torch.tensor([0, *np.cumsum(new)], dtype=torch.int32),
         "lengths": torch.tensor(lengths, dtype=torch.int32)}
    cache = (pages, case["kv_heads"], case["page"], case["dim"])
    half = HALF[case["kind"]]
    t["k"] = [_normal(g, *cache).to(half) for _ in layers]
    t["v"] = [_normal(g, *cache).to(half) for _ in layers]
    if case["op"] == "attend":
        # Scores spread as normalised queries and keys spread them.
        t["q"] = [1.5 * _normal(g, tokens, case["heads"] * case["dim"]) for _ in layers]
        return t
    width = (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    t["qkv"] = [_normal(g, tokens, width) for _ in layers]  # one product's rows: queries, keys, values
    t["q_norm"] = [1 + 0.1 * _normal(g, case["dim"]) for _ in layers]
    t["k_norm"] = [1 + 0.1 * _normal(g, case["dim"]) for _ in layers]
    t["positions"], t["freqs"] = _positions(case, tokens, seed), _freqs(case["rotary"])
    return t


def _freqs(rotary: int) -> torch.Tensor:
    return (1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float()


def _pack_k(k: torch.Tensor) -> torch.Tensor:
    """[page][head][slot][dim] -> blocks of 32 keys, [dim / 8][key order][8]."""
    p, h, n, d = k.shape
    # slot = 32 * block + 8 * a + 4 * b + c is key 16 * b + 4 * a + c of its block.
    return k.view(p, h, n // 32, 4, 2, 4, d // 8, 8).permute(0, 1, 2, 6, 4, 3, 5, 7).contiguous()


def _unpack_k(k: torch.Tensor, shape: tuple) -> torch.Tensor:
    p, h, n, d = shape
    return k.view(p, h, n // 32, d // 8, 2, 4, 4, 8).permute(0, 1, 2, 5, 4, 6, 3, 7).reshape(shape)


def _pack_v(v: torch.Tensor) -> torch.Tensor:
    """[page][head][slot][dim] -> blocks of 32 keys, [key / 8][dim][8]."""
    p, h, n, d = v.shape
    return v.view(p, h, n // 8, 8, d).transpose(3, 4).contiguous()


def _unpack_v(v: torch.Tensor, shape: tuple) -> torch.Tensor:
    p, h, n, d = shape
    return v.view(p, h, n // 8, d, 8).transpose(3, 4).reshape(shape)


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


def _bytes(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous().cpu()
    return t.view(torch.int16) if t.dtype in HALF.values() else t


class DeviceOutputs(dict):
    """Output buffers by name. They stay on the device; looking at one copies
    it to the host."""

    def __getitem__(self, name):
        buffer, shape, kind, unpack = super().__getitem__(name)
        if kind is None:
            return buffer.read(np.float32, math.prod(shape)).reshape(shape)
        raw = torch.from_numpy(buffer.read(np.int16, math.prod(shape))).view(HALF[kind])
        return unpack(raw, shape)


def prepare(case: dict, seed: int) -> dict:
    t = _inputs(case, seed)
    scale = 1 / math.sqrt(case["dim"])
    if not own:
        def put(v):
            return [put(x) for x in v] if isinstance(v, list) else v.cpu().cuda() if isinstance(v, torch.Tensor) else v

        return {"case": case, "scale": scale, **{k: put(v) for k, v in t.items()}}
    gpu, q = _gpu(), _qmr()
    dim, tokens, heads = case["dim"], t["tokens"], case["heads"]
    calls, out = [], {}

    def up(v):
        return gpu.upload_bytes(_bytes(v).numpy())

    def call(name, buffers, params, offsets=None):
        calls.append((name, buffers, params, q.dispatch_layout(name, params)[1], offsets))

    shared = {k: up(t[k]) for k in ("positions", "freqs", "starts", "lengths", "table") if k in t}
    for i in range(case["layers"]):
        if case["op"] == "rope":
            y = gpu.alloc_f32(tokens * heads * dim)
            call("rope_axes", [up(t["x"][i]), shared["positions"], shared["freqs"], y],
                 [tokens, heads, dim, case["rotary"], heads * dim, heads * dim, int(case["adjacent"]),
                  int(case["dealt"]), case["axes"], *_sections(case["rotary"], case["axes"])])
            out["y%d" % i] = (y, (tokens, heads, dim), None, None)
            continue
        kv, page, pages, columns = case["kv_heads"], case["page"], t["pages"], t["table"].shape[1]
        cache = (pages, kv, page, dim)
        kc, vc = up(_pack_k(t["k"][i])), up(_pack_v(t["v"][i]))
        y = gpu.alloc_f32(tokens * heads * dim)
        if case["op"] == "append":
            width = (heads + 2 * kv) * dim
            qkv = up(t["qkv"][i])
            call("kv_append_rope_" + case["kind"],
                 [qkv, qkv, qkv, up(t["q_norm"][i]), up(t["k_norm"][i]), shared["positions"], shared["freqs"],
                  shared["starts"], shared["lengths"], shared["table"], kc, vc, y],
                 [case["batch"], tokens, heads, kv, dim, case["rotary"], width, width, width, heads * dim,
                  int(case["adjacent"]), int(case["dealt"]), case["axes"], *_sections(case["rotary"], case["axes"]),
                  _word(EPS) if case["norm"] else 0, page, pages, columns],
                 [0, 4 * heads * dim, 4 * (heads + kv) * dim] + [0] * 10)
            out["k%d" % i] = (kc, cache, case["kind"], _unpack_k)
            out["v%d" % i] = (vc, cache, case["kind"], _unpack_v)
            out["q%d" % i] = (y, (tokens, heads, dim), None, None)
        else:
            call("attn_paged_" + case["kind"],
                 [up(t["q"][i]), shared["starts"], shared["lengths"], shared["table"], kc, vc, y],
                 [case["batch"], tokens, heads, kv, dim, heads * dim, heads * dim, page, pages, columns, t["longest"],
                  1, case["window"], _word(scale)])
            out["o%d" % i] = (y, (tokens, heads, dim), None, None)
    return {"calls": calls, "out": out}


def run(state: dict):
    if not own:
        return _plain(state)
    command = _gpu().begin()
    for name, buffers, params, threads, offsets in state["calls"]:
        command.encode(name, buffers, params, threads, 64, offsets)
    command.finish()
    command.release()
    return DeviceOutputs(state["out"])


# ---- the plain form: elementary operations in 32 bits ----

def _plain(s: dict) -> dict:
    form = {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[s["case"]["op"]]
    return {k: v for i in range(s["case"]["layers"]) for k, v in form(s, i).items()}


def _turn(x: torch.Tensor, s: dict) -> torch.Tensor:
    """x [tokens][heads][dim], its first `rotary` dimensions rotated."""
    case = s["case"]
    r = case["rotary"]
    axis = torch.tensor(_axis_of(r, case["axes"], case["dealt"]), device=x.device)
    angle = s["positions"].float()[axis].T * s["freqs"]  # [tokens][pairs]
    c, w = angle.cos().unsqueeze(1), angle.sin().unsqueeze(1)
    if case["adjacent"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * w, b * c + a * w], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * c - b * w, b * c + a * w], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_rope(s: dict, i: int) -> dict:
    case = s["case"]
    return {"y%d" % i: _turn(s["x"][i].view(s["tokens"], case["heads"], case["dim"]), s)}


def _rms(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + EPS) * w


def _places(s: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """(sequence, position in its cache) of every new token."""
    starts = s["starts"].long()
    t = torch.arange(s["tokens"], device=starts.device)
    seq = torch.searchsorted(starts, t, right=True) - 1
    new = starts[1:] - starts[:-1]
    return seq, t - starts[seq] + s["lengths"].long()[seq] - new[seq]


def _plain_append(s: dict, i: int) -> dict:
    case = s["case"]
    heads, kv = case["heads"], case["kv_heads"]
    rows = s["qkv"][i].view(s["tokens"], heads + 2 * kv, case["dim"])
    q, k, v = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
    if case["norm"]:
        q, k = _rms(q, s["q_norm"][i]), _rms(k, s["k_norm"][i])
    q, k = _turn(q, s), _turn(k, s)
    seq, at = _places(s)
    page = s["table"].long()[seq, at // case["page"]]
    kc, vc = s["k"][i], s["v"][i]
    kc[page, :, at % case["page"]] = k.to(kc.dtype)
    vc[page, :, at % case["page"]] = v.to(vc.dtype)
    return {"q%d" % i: q, "k%d" % i: kc, "v%d" % i: vc}


def _plain_attend(s: dict, i: int) -> dict:
    case = s["case"]
    heads, kv, dim, batch, page = case["heads"], case["kv_heads"], case["dim"], case["batch"], case["page"]
    longest, new = s["longest"], s["longest_new"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    count = starts[1:] - starts[:-1]
    # Every sequence's queries and pages, padded to the longest.
    slot = torch.arange(new, device=starts.device)
    token = (starts[:-1, None] + slot).clamp(max=s["tokens"] - 1)
    q = s["q"][i].view(-1, kv, heads // kv, dim)[token]  # [batch][new][kv][group][dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(batch * kv, -1, dim)
    columns = -(-longest // page)
    pages = s["table"].long()[:, :columns]
    k = s["k"][i][pages].transpose(1, 2).reshape(batch * kv, columns * page, dim)[:, :longest].float()
    v = s["v"][i][pages].transpose(1, 2).reshape(batch * kv, columns * page, dim)[:, :longest].float()
    at = slot + (lengths - count)[:, None]  # [batch][new]
    key = torch.arange(longest, device=starts.device)
    seen = (key <= at[..., None]) & (key < lengths[:, None, None])
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    score = torch.bmm(q, k.transpose(1, 2)) * s["scale"]
    score = score.view(batch, heads, new, longest).masked_fill(~seen[:, None], -math.inf)
    weight = (score - score.amax(dim=-1, keepdim=True)).exp()
    out = torch.bmm(weight.view(batch * kv, -1, longest), v).view(batch, heads, new, dim)
    out = out / weight.sum(dim=-1, keepdim=True)
    seq, place = _places(s)
    return {"o%d" % i: out[seq, :, place - (lengths - count)[seq]]}


# ---- what a pass cannot do without ----

def work(case: dict) -> dict:
    layers, dim, heads = case["layers"], case["dim"], case["heads"]
    if case["op"] == "rope":
        n = case["tokens"] * heads * dim
        return {"bytes": layers * 8.0 * n + 4 * case["axes"] * case["tokens"],
                "flops": layers * 3.0 * case["tokens"] * heads * case["rotary"]}
    new, lengths = _lengths(case)
    tokens, kv = sum(new), case["kv_heads"]
    if case["op"] == "append":
        return {"bytes": layers * tokens * dim * (8.0 * heads + 2 * 6 * kv),
                "flops": layers * tokens * (heads + kv) * (3.0 * case["rotary"] + (4 * dim if case["norm"] else 0))}
    seen = read = 0
    for n, length in zip(new, lengths):
        first = length - n  # the first new token's position
        w = case["window"] or length
        seen += sum(min(p + 1, w) for p in range(first, length))
        read += length - max(0, first + 1 - w)
    return {"bytes": layers * (8.0 * tokens * heads * dim + 4.0 * read * kv * dim),
            "flops": layers * 4.0 * dim * heads * seen}


# ---- from the definition, in 64 bits ----

def exact(case: dict, seed: int):
    t = _inputs(case, seed)
    out = {}
    for i in range(case["layers"]):
        if case["op"] == "rope":
            x = t["x"][i].view(t["tokens"], case["heads"], case["dim"])
            out["y%d" % i] = _turn64(x.double(), t, case)
        elif case["op"] == "append":
            out.update(_append64(t, case, i))
        else:
            out["o%d" % i] = _attend64(t, case, i)
    return out


def _turn64(x: torch.Tensor, t: dict, case: dict) -> torch.Tensor:
    """Complex multiplication by exp(i * position * frequency)."""
    r = case["rotary"]
    axis = _axis_of(r, case["axes"], case["dealt"])
    angle = t["positions"].double()[axis, :].T * t["freqs"].double()
    turn = torch.polar(torch.ones_like(angle), angle).to(x.device)[:, None, :]
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["adjacent"] else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., first], x[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _append64(t: dict, case: dict, i: int) -> dict:
    heads, kv, page = case["heads"], case["kv_heads"], case["page"]
    rows = t["qkv"][i].view(t["tokens"], heads + 2 * kv, case["dim"]).double()
    q, k, v = rows.split([heads, kv, kv], dim=1)
    if case["norm"]:
        q = q / (q.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * t["q_norm"][i].double()
        k = k / (k.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * t["k_norm"][i].double()
    q, k = _turn64(q, t, case), _turn64(k, t, case)
    kc, vc = t["k"][i].double(), t["v"][i].double()
    starts, lengths, table = t["starts"].tolist(), t["lengths"].tolist(), t["table"]
    for b in range(case["batch"]):
        n = starts[b + 1] - starts[b]
        at = torch.arange(lengths[b] - n, lengths[b])
        pages, slots = table[b].long()[at // page], at % page
        kc[pages, :, slots] = k[starts[b]:starts[b + 1]]
        vc[pages, :, slots] = v[starts[b]:starts[b + 1]]
    return {"q%d" % i: q, "k%d" % i: kc, "v%d" % i: vc}


def _attend64(t: dict, case: dict, i: int) -> torch.Tensor:
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = heads // kv
    q = t["q"][i].view(t["tokens"], heads, dim)
    out = torch.zeros(t["tokens"], heads, dim, dtype=torch.float64, device=q.device)
    starts, lengths = t["starts"].tolist(), t["lengths"].tolist()
    for b in range(case["batch"]):
        length = lengths[b]
        pages = t["table"][b].long()[:-(-length // page)].to(q.device)
        at = torch.arange(length - (starts[b + 1] - starts[b]), length, device=q.device)[:, None]
        key = torch.arange(length, device=q.device)
        seen = key <= at
        if case["window"]:
            seen &= key > at - case["window"]
        for h in range(heads):
            k = t["k"][i][pages, h // group].reshape(-1, dim)[:length].double()
            v = t["v"][i][pages, h // group].reshape(-1, dim)[:length].double()
            rows = slice(starts[b], starts[b + 1])
            score = q[rows, h].double() @ k.T.contiguous() / math.sqrt(dim)
            out[rows, h] = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1) @ v
    return out
