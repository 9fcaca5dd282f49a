"""Performance cases of the operators around a long, mixed text-and-image context: rotary positions with
several axes, a key/value cache held in 8 bits with a scale for each block of tokens and head, the
attention that reads it, the attention weight its tokens accumulate, and eviction by that weight.

Kinds of case (`case["kind"]`):
  rope     F.rope_axes of queries (B, H, S, D), forward, or forward and backward (`train`)
  append   a prompt into an empty 8-bit cache, and the values that the cache then stands for
  attend   attention of the last L tokens' queries over a cache of S tokens (L = 1: a decode step)
  session  clear, append a prompt with rotated keys, then decode steps of one token (append, attend)
  weights  `attend` that also leaves the sum of each token's attention weights
  evict    a prompt into an empty cache, then all but `keep` tokens of each head out by given weights

With `own` false `run` computes the operators from elementary torch operations in float32 (angles in
float64); with `own` true it makes a user's calls of this package.  `exact` is the definition in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
# the largest value of an 8-bit type: its fraction in [0.5, 1) and its exponent, for the block scale
LIMIT = {"int8": (127 / 128, 7), "e4m3": (448 / 512, 9)}


def _case(name, kind, dtype, B, H, Hkv, L, S, D, cache="int8", block=32, train=False, sections=(), interleaved=False,
          steps=0, keep=0, recent=0):
    return {"name": name, "kind": kind, "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "L": L, "S": S, "D": D, "cache": cache,
            "block": block, "train": train, "sections": ",".join(map(str, sections)), "interleaved": interleaved,
            "steps": steps, "keep": keep, "recent": recent}


def listed():
    return [
        # the queries of one decode step of a small batch: latency is all of it
        _case("rope_step_bf16", "rope", "bf16", 4, 32, 32, 0, 1, 128, sections=(16, 24, 24)),
        # the queries of a training batch of text and images, forward and backward, an odd length
        _case("rope_train_bf16", "rope", "bf16", 4, 32, 32, 0, 2047, 128, train=True, sections=(24, 20, 20), interleaved=True),
        # a batch's prompt into an 8-bit cache, the last block not full
        _case("append_int8", "append", "fp16", 4, 32, 8, 0, 2001, 128),
        # a generation session: launches and host work count
        _case("session_e4m3", "session", "bf16", 4, 32, 8, 1, 500, 128, cache="e4m3", steps=8, sections=(16, 24, 24)),
        # one decode step of a serving batch with long contexts, grouped-query
        _case("decode_int8_fp16", "attend", "fp16", 16, 32, 8, 1, 8192, 128),
        # the same of a smaller batch, the other 8-bit type, an odd length
        _case("decode_e4m3_bf16", "attend", "bf16", 4, 32, 8, 1, 3001, 128, cache="e4m3"),
        # the tokens that a draft proposed, checked in one step
        _case("verify_int8_bf16", "attend", "bf16", 8, 32, 8, 5, 4096, 128, block=64),
        # a chunk of a prompt over what the cache holds of it
        _case("chunk_int8_fp16", "attend", "fp16", 4, 32, 8, 500, 1500, 128),
        # the last tokens of a prompt observed, to see which others they attend to
        _case("window_int8_fp16", "weights", "fp16", 4, 32, 8, 32, 4096, 128),
        # a decode step on an ordinary cache that keeps count of its tokens' weights
        _case("weights_fp16", "weights", "fp16", 4, 32, 8, 1, 4096, 128, cache="fp16"),
        # half of a prompt's tokens leave an 8-bit cache
        _case("evict_int8", "evict", "fp16", 4, 32, 8, 0, 4096, 128, keep=2048, recent=64),
        # two thirds leave an ordinary cache of one sequence, odd sizes
        _case("evict_bf16", "evict", "bf16", 1, 8, 8, 0, 3001, 64, cache="bf16", keep=1000, recent=33),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, pairs, interleaved):
    """Pairs of each axis: time, height, width."""
    side = rng.randint(max(1, pairs // 5), pairs // 3)
    if interleaved:
        side = min(side, (pairs - 2) // 3)
    return (pairs - 2 * side, side, side)


def draw(rng):
    kind = rng.choice(["rope", "rope", "append", "session", "attend", "attend", "attend", "weights", "weights", "evict"])
    dtype = rng.choice(["fp16", "bf16", "bf16", "fp32"])
    D = rng.choice([64, 128, 128, 80])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 2, 4, 7])
    block = rng.choice([32, 32, 64, 128])
    cache = rng.choice(["int8", "int8", "e4m3"])
    if kind == "rope":
        mixed = rng.random() < 0.5
        H, S = rng.choice([4, 8, 14, 32]), _log(rng, 1, 2047)
        most = int(4 * 32 * 2047 * 128 * 2 / (H * S * D * SIZE[dtype]))
        return _trim(_case("", kind, dtype, _log(rng, 1, max(1, min(8, most))), H, H, 0, S, D, train=rng.random() < 0.5,
                           sections=_split(rng, D // 2, mixed), interleaved=mixed))
    if kind == "append":
        S = _log(rng, 16, 2001)
        most = int(4 * 8 * 2001 * 128 * 2 / (Hkv * S * D * SIZE[dtype]))
        return _trim(_case("", kind, dtype, _log(rng, 1, max(1, min(8, most))), H, Hkv, 0, S, D, cache, block))
    if kind == "session":
        return _trim(_case("", kind, rng.choice(["fp16", "bf16"]), rng.randint(1, 4), H, Hkv, 1, _log(rng, 20, 500), D, cache, block,
                           steps=rng.randint(2, 8), sections=_split(rng, D // 2, False)))
    if kind == "attend":
        L = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 16, 500)])
        if L == 1:
            S = _log(rng, 1, 8192)
            most = 16 * 8 * 8192 // (Hkv * S)
        elif L <= 8:
            S = _log(rng, L, 4096)
            most = 8 * 8 * 4096 // (Hkv * S)
        else:
            S = L + _log(rng, 1, 1000)
            most = 4 * 32 * 500 * 1500 // (H * L * S * (2 if dtype == "fp32" else 1))
        return _trim(_case("", kind, dtype, _log(rng, 1, max(1, min(16, most))), H, Hkv, L, S, D, cache, block))
    if kind == "weights":
        L = rng.choice([1, 1, _log(rng, 2, 32)])
        S = _log(rng, max(L, 32), 4096)
        most = 4 * 8 * 4096 // (Hkv * S)
        return _trim(_case("", kind, dtype, _log(rng, 1, max(1, min(8, most))), H, Hkv, L, S, D,
                           rng.choice(["int8", "e4m3", dtype]), block))
    S = _log(rng, 64, 4096)
    most = int(4 * 8 * 4096 * 128 * 2 / (Hkv * S * D * SIZE[dtype]))
    keep = _log(rng, 16, S)
    return _trim(_case("", kind, dtype, _log(rng, 1, max(1, min(8, most))), H, Hkv, 0, S, D,
                       rng.choice(["int8", "e4m3", dtype]), block, keep=keep, recent=rng.randint(0, keep // 2)))


def _trim(case):
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------------------


def _sections(case):
    return tuple(int(x) for x in case["sections"].split(","))


def _positions(case, seed, n):
    """Positions (3, B, n): text, where the axes move together, and in it an image, whose time stands still
    while height and width run over its patches; the context starts anywhere in a long one."""
    gen = torch.Generator().manual_seed(seed + 5)
    pos = torch.empty((3, case["B"], n), dtype=torch.int64)
    for b in range(case["B"]):
        start = int(torch.randint(0, 60000, (), generator=gen))
        head = int(torch.randint(0, n // 4 + 1, (), generator=gen))
        side = int(math.isqrt(n // 2))
        i = torch.arange(side * side)
        text = torch.arange(n - head - side * side) + start + head + side
        for a, image in enumerate((torch.zeros_like(i), i // max(side, 1), i % max(side, 1))):
            pos[a, b] = torch.cat([torch.arange(head) + start, image + start + head, text])
    return pos


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, H, Hkv, L, S, D = (case[n] for n in ("B", "H", "Hkv", "L", "S", "D"))
    dt = DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "rope":
        t = {"x": _normal(gen, (B, H, S, D), dt), "pos": _positions(case, seed, S).to(DEV)}
        if case["train"]:
            t["dout"] = _normal(gen, (B, H, S, D), dt)
        return t
    n = S + case["steps"]
    # keys differ in size between their dimensions, as projected keys do
    size = 0.5 + torch.rand((1, Hkv, 1, D), generator=gen, device=DEV) * 1.5
    t = {"k": (_normal(gen, (B, Hkv, n, D), torch.float32) * size).to(dt), "v": _normal(gen, (B, Hkv, n, D), dt)}
    if kind == "session":
        t["q"] = _normal(gen, (B, H, case["steps"], D), dt)
        t["pos"] = _positions(case, seed, n).to(DEV)
    elif kind in ("attend", "weights"):
        t["q"] = _normal(gen, (B, H, L, D), dt)
    elif kind == "evict":
        # a few tokens take most of the weight; 2^-12 apart at the least, so that some are equal
        w = torch.rand((B, Hkv, S), generator=gen, device=DEV) ** 4
        t["weights"] = torch.round(w * 4096) / 4096
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, **t}
    kind = case["kind"]
    if kind == "rope":
        state["sections"] = _sections(case)
        if own and case["train"]:
            state["x"] = t["x"].requires_grad_()
        return state
    if kind == "session":
        state["sections"] = _sections(case)
    cap = case["S"] + case["steps"]
    if own:
        from gguf_train_amd import KVCache

        dtypes = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, **DTYPES}
        blocks = {"block_tokens": case["block"]} if case["cache"] in LIMIT else {}
        cache = KVCache(case["B"], case["Hkv"], cap, case["D"], dtypes[case["cache"]], DEV, **blocks)
    else:
        cache = _Cache(case)
    if kind in ("attend", "weights"):
        cache.append(state.pop("k"), state.pop("v"))
    state["cache"] = cache
    return state


# ---- the plain forms ------------------------------------------------------------------------------


def _axes(sections, interleaved, device):
    """The axis of each pair: the sections one after the other, or one pair of each axis in turn while an axis
    past the first has pairs left."""
    n = len(sections)
    if not interleaved:
        return torch.tensor([a for a in range(n) for _ in range(sections[a])], device=device)
    return torch.tensor([i % n if i // n < sections[i % n] else 0 for i in range(sum(sections))], device=device)


def _turn(x, pos, sections, interleaved, sign=1.0):
    """x (B, H, S, D) rotated in float32 by angles of float64: pairs (i, i + D/2)."""
    half = x.shape[-1] // 2
    freq = 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = pos[_axes(sections, interleaved, x.device)].permute(1, 2, 0).double() * freq  # (B, S, half)
    c, s = angle.cos().float()[:, None], (sign * angle.sin()).float()[:, None]
    lo, hi = x[..., :half].float(), x[..., half:].float()
    return torch.cat([lo * c - hi * s, lo * s + hi * c], -1).to(x.dtype)


def _quantise(x, kind):
    """Codes and scales of blocks x (..., N, D), the last two dimensions sharing a scale: the power of two that
    puts the largest magnitude just within the 8-bit type."""
    fraction, exponent = LIMIT[kind]
    amax = x.abs().amax((-2, -1), keepdim=True)
    m, e = torch.frexp(amax)
    e = e - exponent + (m > fraction).int()
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(amax), e)
    y = x / scale
    codes = torch.round(y).to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
    return codes, scale


class _Cache:
    """What a program without the package would keep: codes and scales of whole blocks and the tokens after
    them, or (cache dtype of the inputs) the tokens."""

    def __init__(self, case):
        self.case, self.kind, self.block = case, case["cache"], case["block"]
        self.clear()

    def clear(self):
        B, Hkv, D = (self.case[n] for n in ("B", "Hkv", "D"))
        dt = torch.float32 if self.kind in LIMIT else DTYPES[self.kind]
        self.codes = {n: None for n in "kv"}
        self.scales = {n: None for n in "kv"}
        self.tail = {n: torch.empty((B, Hkv, 0, D), device=DEV, dtype=dt) for n in "kv"}

    def append(self, k, v):
        for n, new in (("k", k), ("v", v)):
            x = torch.cat([self.tail[n], new.to(self.tail[n].dtype)], 2)
            if self.kind in LIMIT:
                B, Hkv, T, D = x.shape
                full = T // self.block * self.block
                if full:
                    codes, scale = _quantise(x[:, :, :full].reshape(B, Hkv, full // self.block, self.block, D), self.kind)
                    old = self.codes[n]
                    self.codes[n] = codes if old is None else torch.cat([old.view(torch.uint8), codes.view(torch.uint8)], 2).view(old.dtype)
                    self.scales[n] = scale if old is None else torch.cat([self.scales[n], scale], 2)
                    x = x[:, :, full:]
            self.tail[n] = x

    def values(self, n):
        if self.codes[n] is None:
            return self.tail[n].float()
        x = self.codes[n].float() * self.scales[n]
        return torch.cat([x.flatten(2, 3), self.tail[n]], 2)

    def attend(self, q, weights=False):
        k, v = self.values("k"), self.values("v")
        B, H, L, D = q.shape
        Hkv, S = k.shape[1], k.shape[2]
        s = torch.matmul(q.float().reshape(B, Hkv, -1, D), k.transpose(2, 3)) / math.sqrt(D)
        s = s.reshape(B, H, L, S)
        if L > 1:
            late = torch.arange(S, device=DEV)[None, :] > torch.arange(S - L, S, device=DEV)[:, None]
            s = s.masked_fill(late, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out = torch.matmul(p.reshape(B, Hkv, -1, S), v).reshape(B, H, L, D).to(q.dtype)
        return (out, p.reshape(B, Hkv, -1, S).sum(2)) if weights else out


def _chosen(weights, keep, recent):
    """Per head, the `recent` last tokens and those of the largest weights among the others (the first of equal
    ones), in order."""
    B, Hkv, S = weights.shape
    if S <= keep:
        kept = torch.arange(S, device=DEV).expand(B, Hkv, S)
        return torch.cat([kept, torch.full((B, Hkv, keep - S), -1, device=DEV)], 2)
    order = torch.sort(weights[..., :S - recent], dim=-1, descending=True, stable=True).indices[..., :keep - recent]
    last = torch.arange(S - recent, S, device=DEV).expand(B, Hkv, recent)
    return torch.cat([order.sort(-1).values, last], -1)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "rope":
        y = _turn(state["x"], state["pos"], state["sections"], case["interleaved"])
        if not case["train"]:
            return y
        return y, _turn(state["dout"], state["pos"], state["sections"], case["interleaved"], -1.0)
    cache = state["cache"]
    if kind == "attend":
        return cache.attend(state["q"])
    if kind == "weights":
        return cache.attend(state["q"], True)
    k, v, S = state["k"], state["v"], case["S"]
    cache.clear()
    if kind == "session":
        pos, sec = state["pos"], state["sections"]
        cache.append(_turn(k[:, :, :S], pos[..., :S], sec, False), v[:, :, :S])
        out = []
        for i in range(S, S + case["steps"]):
            at = pos[..., i:i + 1]
            cache.append(_turn(k[:, :, i:i + 1], at, sec, False), v[:, :, i:i + 1])
            out.append(cache.attend(_turn(state["q"][:, :, i - S:i - S + 1], at, sec, False)))
        return out
    cache.append(k, v)
    if kind == "append":
        return cache.values("k"), cache.values("v")
    kept = _chosen(state["weights"], case["keep"], case["recent"])
    rows = kept[..., :min(case["keep"], S)][..., None].expand(-1, -1, -1, case["D"])
    left = [torch.gather(cache.values(n), 2, rows) for n in "kv"]
    if S > case["keep"]:
        cache.clear()
        cache.append(*left)
    return kept, cache.values("k"), cache.values("v")


def run(state):
    if not own:
        return _plain(state)
    from gguf_train_amd.nn import functional as F

    case = state["case"]
    kind = case["kind"]
    if kind == "rope":
        y = F.rope_axes(state["x"], state["pos"], state["sections"], interleaved=case["interleaved"])
        if not case["train"]:
            return y
        return y, torch.autograd.grad(y, state["x"], state["dout"])[0]
    cache = state["cache"]
    if kind == "attend":
        return cache.attention(state["q"])
    if kind == "weights":
        out = cache.attention(state["q"], accumulate=0.0)
        return out, cache.weights()
    k, v, S = state["k"], state["v"], case["S"]
    cache.clear()
    if kind == "session":
        pos, sec = state["pos"], state["sections"]
        cache.append(k[:, :, :S], v[:, :, :S], rope={"positions": pos[..., :S], "sections": sec, "mode": 2})
        out = []
        for i in range(S, S + case["steps"]):
            at = pos[..., i:i + 1]
            cache.append(k[:, :, i:i + 1], v[:, :, i:i + 1], rope={"positions": at, "sections": sec, "mode": 2})
            out.append(cache.attention(F.rope_axes(state["q"][:, :, i - S:i - S + 1], at, sec)))
        return out
    cache.append(k, v)
    if kind == "append":
        return cache.read()
    kept = cache.evict(case["keep"], case["recent"], state["weights"])
    return (kept, *cache.read())


# ---- work and definition --------------------------------------------------------------------------


def work(case):
    B, H, Hkv, L, S, D = (case[n] for n in ("B", "H", "Hkv", "L", "S", "D"))
    es, kind = SIZE[case["dtype"]], case["kind"]
    cs = SIZE.get(case["cache"], 1)
    if kind == "rope":
        n = B * H * S * D * (2 if case["train"] else 1)
        return {"bytes": 2 * n * es + 3 * B * S * 8, "flops": 3 * n}
    row = B * Hkv * D
    if kind == "append":
        return {"bytes": 2 * row * S * (es + 2 * cs + 4), "flops": 2 * row * S * 2}
    if kind == "evict":
        keep = min(case["keep"], S)
        return {"bytes": 2 * row * (S * (es + cs) + keep * (3 * cs + 4)) + B * Hkv * (4 * S + 8 * keep), "flops": 2 * row * (S + keep)}
    steps = case["steps"]
    if kind == "session":
        seen = sum(range(S + 1, S + steps + 1))
        return {"bytes": 2 * row * ((S + steps) * (es + cs) + seen * cs) + 2 * B * H * D * steps * es,
                "flops": 4 * B * H * D * seen + 3 * row * (S + steps)}
    pairs = L * S - L * (L - 1) // 2
    more = B * Hkv * S * 4 if kind == "weights" else 0
    return {"bytes": 2 * row * S * cs + 2 * B * H * L * D * es + more, "flops": 4 * B * H * D * pairs}


def _held64(x, case):
    """The values in float64 that a cache of the tokens x (B, Hkv, T, D) stands for."""
    x, kind, N = x.double().clone(), case["cache"], case["block"]
    if kind not in LIMIT:
        return x
    top = {"int8": 127.0, "e4m3": 448.0}[kind]
    for j in range(x.shape[2] // N):
        b = x[:, :, N * j:N * (j + 1)]
        most = b.abs().flatten(2).amax(2)[..., None, None]
        unit = torch.exp2(torch.ceil(torch.log2(most / top)))  # off by one where log2 rounds: put right below
        unit = torch.where(most > top * unit, 2 * unit, unit)
        unit = torch.where(most <= top * unit / 2, unit / 2, unit)
        unit = torch.where(most > 0, unit, torch.ones_like(unit))
        y = b / unit
        if kind == "int8":
            b.copy_(torch.round(y) * unit)
        else:
            # 3 bits after the leading one, down to 2^-6; fixed steps of 2^-9 below
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            b.copy_(torch.round(y / step) * step * unit)
    return x


def _turned64(x, pos, case, back=False):
    half = x.shape[-1] // 2
    sections, i = _sections(case), 0
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    left = list(sections)
    for i in range(half):
        if case["interleaved"]:
            a = i % 3 if i // 3 < sections[i % 3] else 0
        else:
            a = next(n for n in range(3) if left[n] > 0)
            left[a] -= 1
        angle = pos[a].double() * 10000.0 ** (-2.0 * i / (2 * half))
        turn = torch.polar(torch.ones_like(angle), -angle if back else angle)[:, None]
        z = torch.complex(x[..., i].double(), x[..., i + half].double()) * turn
        out[..., i], out[..., i + half] = z.real, z.imag
    return out


def _attend64(q, k, v):
    B, H, L, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    out = torch.empty((B, H, L, D), dtype=torch.float64, device=q.device)
    weights = torch.zeros((B, Hkv, S), dtype=torch.float64, device=q.device)
    seen = torch.arange(S, device=q.device)[None] <= torch.arange(S - L, S, device=q.device)[:, None]
    for b in range(B):
        for h in range(H):
            g = h // (H // Hkv)
            s = (q[b, h].double() @ k[b, g].T) / math.sqrt(D)
            p = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), 1)
            out[b, h] = p @ v[b, g]
            weights[b, g] += p.sum(0)
    return out, weights


def exact(case, seed):
    t = _inputs(case, seed)
    kind, S = case["kind"], case["S"]
    if kind == "rope":
        y = _turned64(t["x"], t["pos"], case)
        return (y, _turned64(t["dout"], t["pos"], case, True)) if case["train"] else y
    k, v = t["k"], t["v"]
    if kind == "append":
        return _held64(k, case), _held64(v, case)
    if kind in ("attend", "weights"):
        out, weights = _attend64(t["q"], _held64(k, case), _held64(v, case))
        return (out, weights) if kind == "weights" else out
    if kind == "session":
        # rotated keys and queries are held in the inputs' type
        k = _turned64(k, t["pos"], case).to(k.dtype)
        q = _turned64(t["q"], t["pos"][..., S:], case).to(k.dtype)
        out = []
        for i in range(case["steps"]):
            n = S + i + 1
            out.append(_attend64(q[:, :, i:i + 1], _held64(k[:, :, :n], case), _held64(v[:, :, :n], case))[0])
        return out
    K, V = _held64(k, case), _held64(v, case)
    keep, recent = case["keep"], case["recent"]
    if S <= keep:
        kept = torch.full((case["B"], case["Hkv"], keep), -1, dtype=torch.int64, device=k.device)
        kept[..., :S] = torch.arange(S, device=k.device)
        return kept, K, V
    kept, rows = torch.empty((case["B"], case["Hkv"], keep), dtype=torch.int64), {"k": [], "v": []}
    w = t["weights"].cpu().tolist()
    for b in range(case["B"]):
        for g in range(case["Hkv"]):
            first = sorted(range(S - recent), key=lambda i: (-w[b][g][i], i))[:keep - recent]
            kept[b, g] = torch.tensor(sorted(first) + list(range(S - recent, S)))
            at = kept[b, g].to(k.device)
            rows["k"].append(K[b, g, at])
            rows["v"].append(V[b, g, at])
    shape = (case["B"], case["Hkv"], keep, case["D"])
    left = [torch.stack(rows[n]).reshape(shape) for n in "kv"]
    return (kept.to(k.device), *(_held64(x, case) for x in left))
