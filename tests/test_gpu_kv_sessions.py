"""Sessions on block caches in random order: appends, clears, attention, counting of weights and eviction, on
sequences whose lengths part, against a float64 mirror of what the cache should hold."""

import random

import pytest
import torch

import gguf_train_amd as g

import _kv_ref as ref
from _util import randn

pytestmark = pytest.mark.gpu


class Mirror:
    """The tokens of every sequence, as they came or (whole blocks, after an eviction) as they were held."""

    def __init__(self, B, Hkv, D, kind, block):
        self.kind, self.block = kind, block
        self.k = [torch.zeros((Hkv, 0, D), dtype=torch.float64) for _ in range(B)]
        self.v = [x.clone() for x in self.k]
        self.position = [0] * B

    def held(self, b):
        return tuple(ref.held(x, self.kind, self.block) if x.shape[1] else x for x in (self.k[b], self.v[b]))


@pytest.mark.parametrize("seed", [*range(20), 94])
def test_session(dev, seed):
    rng = random.Random(1000 + seed)
    kind, dtype = rng.choice([torch.int8, torch.float8_e4m3fn]), rng.choice([torch.float16, torch.bfloat16, torch.float32])
    block, D = rng.choice([32, 64, 128]), rng.choice([1, 17, 48, 64, 80, 128, 200, 256])
    B, Hkv, G, cap = rng.randint(1, 4), rng.randint(1, 3), rng.choice([1, 2, 3, 7, 16]), rng.choice([150, 256, 700])
    c = g.KVCache(B, Hkv, cap, D, kind, dev, block_tokens=block)
    m = Mirror(B, Hkv, D, kind, block)
    n = seed * 1000
    for step in range(14):
        n += 10
        room, shortest = cap - max(c.lengths), min(c.lengths)
        op = rng.choice(["append", "append", "attend", "count", "evict", "clear"])
        what = (seed, step, op, c.lengths)
        if op == "append" and room > 0:
            T = min(room, rng.choice([1, 1, 2, 5, 31, 33, 64, 100, 130, 400]))
            k, v = randn((B, Hkv, T, D), n, dtype), randn((B, Hkv, T, D), n + 1, dtype) * 2.0 ** rng.randint(-9, 9)
            c.append(k.to(dev), v.to(dev))
            for b in range(B):
                m.k[b], m.v[b] = torch.cat([m.k[b], k[b].double()], 1), torch.cat([m.v[b], v[b].double()], 1)
                m.position[b] += T
        elif op in ("attend", "count") and shortest > 0:
            L, causal = min(shortest, rng.choice([1, 1, 2, 5, 17, 90])), rng.random() < 0.8
            q = randn((B, G * Hkv, L, D), n + 2, dtype)
            before = c.weights().double().cpu() if op == "count" else None
            got = c.attention(q.to(dev), is_causal=causal, accumulate=0.5 if op == "count" else None).double().cpu()
            for b in range(B):
                K, V = m.held(b)
                out, mass, slack, sums, sums_slack = ref.attend(q[b], K, V, causal)
                # A tail's element x enters as y = x / 2^e, |y| < 2 for the row's largest, in float16 hi + lo: hi leaves
                # 2^-11 |y|, or 2^-25 where float16's steps are the least, 2^-24; lo leaves 2^-11 of that, or again
                # 2^-25.  The first is within `bounds`, the second is 2^-25 of the row's largest element at most.
                tail = V[:, K.shape[1] // block * block:]
                least = 2.0 ** -25 * tail.abs().max().item() if tail.shape[1] else 0.0
                off, bound = (got[b] - out).abs(), ref.bounds(out, mass, slack, K.shape[1], dtype) + least
                assert (off <= bound).all(), (what, b, (off - bound).max().item())
                if op == "count":
                    now, want = c.weights()[b].double().cpu(), 0.5 * before[b, :, :K.shape[1]] + sums
                    # p and its log-sum-exp each off by a slack, the exponential's own 2^-22, float32 sums over the rows
                    tol = 2 * sums_slack + (sums + want) * (G * L + 64) * 2.0 ** -24 + sums * 2.0 ** -20 + 1e-37
                    assert ((now[:, :K.shape[1]] - want).abs() <= tol).all(), (what, b)
                    assert not now[:, K.shape[1]:].any()
        elif op == "evict" and max(c.lengths) > 0:
            keep = rng.randint(1, max(c.lengths))
            recent = rng.randint(0, keep)
            w = torch.round(torch.rand((B, Hkv, max(c.lengths)), generator=torch.Generator().manual_seed(n)) * 20) / 20
            before, lengths = c.weights().cpu(), c.lengths
            kept = c.evict(keep, recent, w.to(dev)).cpu()
            for b, held in enumerate(lengths):
                K, V = m.held(b)
                for h in range(Hkv):
                    assert kept[b, h].tolist() == ref.chosen(w[b, h, :held], keep, recent), (what, b, h)
                if held > keep:
                    at = kept[b][..., None].expand(-1, -1, D)
                    m.k[b], m.v[b] = torch.gather(K, 1, at), torch.gather(V, 1, at)
                    now = c.weights()[b].cpu()
                    assert torch.equal(now[:, :keep], torch.gather(before[b], 1, kept[b])) and not now[:, keep:].any()
        elif op == "clear":
            b = rng.randrange(B)
            c.clear(b)
            m.k[b], m.v[b], m.position[b] = m.k[b][:, :0], m.v[b][:, :0], 0
            assert not c.weights()[b].any()
        assert c.lengths == [x.shape[1] for x in m.k] and [c.position(b) for b in range(B)] == m.position
        if max(c.lengths) > 0:
            for got, i in zip(c.read(), range(2)):
                for b in range(B):
                    want, row = m.held(b)[i], got[b].double().cpu()
                    assert torch.equal(row[:, :want.shape[1]], want) and not row[:, want.shape[1]:].any(), (what, b, i)
