"""Accumulated attention weights and eviction on every kind of cache, against float64 and exact selection."""

import math

import pytest
import torch

import gguf_train_amd as g
from gguf_train_amd.nn import functional as F

import _kv_ref as ref
from _util import randn

pytestmark = pytest.mark.gpu

CACHES = [torch.int8, torch.float8_e4m3fn, torch.float16, torch.bfloat16, torch.float32, "q8_0"]


def make(dev, k, v, kind, cap=None, block=32):
    B, Hkv, T, D = k.shape
    c = g.KVCache(B, Hkv, cap or T, D, kind, dev, **({"block_tokens": block} if kind in ref.TOP else {}))
    c.append(k.to(dev), v.to(dev))
    return c


def weight_checks(c, got, q, before, keep, causal, what):
    """`got` = keep * before + the sums over this call's rows, for every sequence; zeros past its length."""
    k = c.read()[0].double().cpu()
    got = got.double().cpu()
    rows = q.shape[1] // k.shape[1] * q.shape[2]
    for b, n in enumerate(c.lengths):
        _, _, _, sums, slack = ref.attend(q[b], k[b, :, :n], k[b, :, :n], causal)
        want = keep * before[b, :, :n] + sums
        # p and its log-sum-exp each off by `slack`, the exponential's own 2^-22, float32 sums over the rows
        tol = slack * 2 + (sums + want) * (rows + 64) * 2.0 ** -24 + sums * 2.0 ** -20 + 1e-37
        assert ((got[b, :, :n] - want).abs() <= tol).all(), (what, b, ((got[b, :, :n] - want).abs() / tol).max().item())
        assert got[b, :, n:].abs().max().item() == 0.0 if got.shape[2] > n else True


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,L,T,D", [(1, 4, 1, 1, 1, 64), (2, 8, 2, 1, 300, 128), (1, 7, 1, 1, 65, 64), (1, 8, 2, 20, 170, 128),
                                           (2, 6, 3, 100, 130, 64), (1, 4, 4, 33, 33, 256), (1, 4, 2, 700, 700, 64), (1, 2, 1, 3, 100, 96)])
def test_weights(dev, kind, dtype, B, H, Hkv, L, T, D):
    k, v, q = randn((B, Hkv, T, D), 1, dtype), randn((B, Hkv, T, D), 2, dtype), randn((B, H, L, D), 3, dtype)
    c = make(dev, k, v, kind, cap=T + 5)
    plain = c.attention(q.to(dev))
    out = c.attention(q.to(dev), accumulate=1.0)
    assert torch.equal(out, plain)
    zero = torch.zeros((B, Hkv, T), dtype=torch.float64)
    first = c.weights().clone()
    weight_checks(c, first, q, zero, 0.0, True, "first")
    q2 = randn((B, H, L, D), 4, dtype)
    c.attention(q2.to(dev), accumulate=0.5, is_causal=False)
    second = c.weights().clone()
    weight_checks(c, second, q2, first.double().cpu(), 0.5, False, "second")
    c.attention(q.to(dev), accumulate=0.0)
    weight_checks(c, c.weights(), q, zero, 0.0, True, "anew")
    assert torch.equal(c.weights(), first)  # (the same bits)


@pytest.mark.parametrize("kind", [torch.int8, torch.float16])
def test_weights_of_ragged_sequences_and_clear(dev, kind):
    B, H, Hkv, D = 3, 4, 2, 64
    k = randn((B, Hkv, 150, D), 5, torch.float16)
    c = make(dev, k, k, kind, cap=200)
    c.attention(randn((B, H, 1, D), 6, torch.float16).to(dev), accumulate=1.0)
    c.clear(1)
    assert c.weights()[1].abs().max().item() == 0.0 and c.weights()[0].sum().item() > 0
    c.append(k[:, :, :40].to(dev), k[:, :, :40].to(dev))
    before = c.weights().double().cpu().clone()
    q = randn((B, H, 5, D), 7, torch.float16)
    c.attention(q.to(dev), accumulate=1.0)
    assert c.lengths == [190, 40, 190]
    weight_checks(c, c.weights(), q, before, 1.0, True, "ragged")
    c.clear()
    assert c.weights().abs().max().item() == 0.0


def test_weights_ignore_what_is_not_finite_elsewhere(dev):
    """A NaN token is met by the rows that see it alone; sums that start anew forget it."""
    for kind in (torch.int8, torch.float32):
        k = randn((1, 1, 70, 64), 8)
        k[0, 0, 69, 3] = math.nan
        c = make(dev, k, randn((1, 1, 70, 64), 9), kind)
        q = randn((1, 2, 3, 64), 10)
        c.attention(q.to(dev), accumulate=1.0)
        w = c.weights()[0, 0]
        if kind == torch.int8:  # (the float caches' kernels give a row with a NaN the log-sum-exp +inf: no weights)
            assert torch.isnan(w[:69]).all()  # the last row's weights
        k2 = randn((1, 1, 70, 64), 11)
        c.clear()
        c.append(k2.to(dev), k2.to(dev))
        c.attention(q.to(dev), accumulate=1.0)
        weight_checks(c, c.weights(), q, torch.zeros((1, 1, 70), dtype=torch.float64), 1.0, True, "afterwards")


def tokens(c):
    return [x.cpu() for x in c.read()]


@pytest.mark.parametrize("kind", CACHES)
@pytest.mark.parametrize("B,Hkv,T,D,keep,recent", [(2, 3, 200, 64, 100, 10), (1, 1, 33, 128, 1, 0), (1, 2, 300, 96, 299, 0), (2, 1, 2500, 64, 1000, 1000),
                                                   (1, 4, 64, 256, 32, 31), (1, 1, 1500, 32, 7, 3), (1, 2, 9001, 32, 700, 9)])
def test_evict(dev, kind, B, Hkv, T, D, keep, recent):
    k, v = randn((B, Hkv, T, D), 20, torch.float16), randn((B, Hkv, T, D), 21, torch.float16)
    c = make(dev, k, v, kind, cap=T + 40)
    w = torch.round(torch.rand((B, Hkv, T)) * 50) / 50  # many equal ones
    old = tokens(c)
    kept = c.evict(keep, recent, w.to(dev)).cpu()
    assert kept.dtype == torch.int64 and c.lengths == [keep] * B and [c.position(b) for b in range(B)] == [T] * B
    for b in range(B):
        for h in range(Hkv):
            assert kept[b, h].tolist() == ref.chosen(w[b, h], keep, recent), (b, h)
    at = kept[..., None].expand(-1, -1, -1, D)
    for got, x in zip(tokens(c), old):
        want = torch.gather(x, 2, at)
        if kind in ref.TOP:
            want = ref.held(want, kind, 32)
        assert torch.equal(got.double(), want.double())
    # and it goes on: new tokens, attention over what stayed and them
    k2, v2, q = randn((B, Hkv, 9, D), 22, torch.float16), randn((B, Hkv, 9, D), 23, torch.float16), randn((B, 2 * Hkv, 3, D), 24, torch.float16)
    c.append(k2.to(dev), v2.to(dev), pos_offset=T)
    got, (K, V) = c.attention(q.to(dev)).double().cpu(), tokens(c)
    for b in range(B):
        out, mass, slack, _, _ = ref.attend(q[b], K[b], V[b])
        tol = ref.bounds(out, mass, slack, keep + 9, torch.float16) if kind in ref.TOP else 2e-3 * out.abs().clamp(min=1) + 2.0 ** -11 * out.abs()
        assert ((got[b] - out).abs() <= tol).all()


@pytest.mark.parametrize("kind", [torch.int8, torch.bfloat16, "q8_0"])
def test_evict_by_accumulated_weights(dev, kind):
    B, H, Hkv, T, D, keep, recent = 2, 4, 2, 180, 64, 64, 8
    k, v = randn((B, Hkv, T, D), 30, torch.bfloat16, 2.0), randn((B, Hkv, T, D), 31, torch.bfloat16)
    c = make(dev, k, v, kind)
    with pytest.raises(RuntimeError, match="no attention weights have been accumulated"):
        c.evict(keep, recent)
    c.attention(randn((B, H, 16, D), 32, torch.bfloat16).to(dev), accumulate=1.0)
    w = c.weights().cpu()
    kept = c.evict(keep, recent).cpu()
    for b in range(B):
        for h in range(Hkv):
            assert kept[b, h].tolist() == ref.chosen(w[b, h], keep, recent)
    assert torch.equal(c.weights().cpu()[..., :keep], torch.gather(w, 2, kept))
    assert c.weights()[..., keep:].abs().max().item() == 0.0
    before = c.weights().double().cpu().clone()
    q = randn((B, H, 2, D), 33, torch.bfloat16)
    c.attention(q.to(dev), accumulate=1.0)
    weight_checks(c, c.weights(), q, before, 1.0, True, "after eviction")


def test_shorter_sequences_are_left_alone(dev):
    for kind in CACHES:
        k = randn((3, 2, 100, 64), 40, torch.float16)
        c = make(dev, k, k, kind, cap=160)
        c.clear(1)
        c.append(k[:, :, :50].to(dev), k[:, :, :50].to(dev))
        old, w = tokens(c), torch.rand((3, 2, 160))
        kept = c.evict(70, 5, w.to(dev)).cpu()
        assert c.lengths == [70, 50, 70] and [c.position(b) for b in range(3)] == [150, 50, 150]
        assert kept[1, 0].tolist() == list(range(50)) + [-1] * 20
        for got, x in zip(tokens(c), old):
            assert torch.equal(got[1, :, :50], x[1, :, :50])
        assert torch.equal(kept, c.evict(70, 5, w.to(dev)).cpu() * 0 + kept)
        # nothing to do: the tokens that are there
        again = c.evict(100, 0, w.to(dev)).cpu()
        assert again[0, 0].tolist() == list(range(70)) + [-1] * 30 and c.lengths == [70, 50, 70]


def test_orders_of_weights(dev):
    """Negative, zero of either sign, infinite and NaN weights; other dtypes and strides; weights on the host."""
    T, keep = 40, 13
    k = randn((1, 1, T, 64), 50)
    w = randn((1, 1, T), 51)
    w[0, 0, 3:6] = torch.tensor([0.0, -0.0, 0.0])
    w[0, 0, 10], w[0, 0, 11], w[0, 0, 12], w[0, 0, 13] = math.inf, -math.inf, math.nan, -math.nan
    for variant in (w, w.double(), w.half(), torch.stack([w, w], -1)[..., 0], w.transpose(0, 1).contiguous().transpose(0, 1)):
        for place in (variant.to(dev), variant):
            c = make(dev, k, k, torch.float16)
            assert c.evict(keep, 2, place).cpu()[0, 0].tolist() == ref.chosen(variant[0, 0].float(), keep, 2)
    c = make(dev, k, k, torch.int8)
    assert c.evict(20, 0, torch.zeros((1, 1, T), device=dev)).cpu()[0, 0].tolist() == list(range(20))


@pytest.mark.parametrize("kind", [torch.float16, torch.int8, "q8_0"])
def test_rope_positions_go_on(dev, kind):
    """One-axis RoPE of tokens appended after an eviction turns by their position, not by their place."""
    T, keep, D = 90, 40, 64
    k, v = randn((2, 2, T, D), 60, torch.float16), randn((2, 2, T, D), 61, torch.float16)
    c = g.KVCache(2, 2, 128, D, kind, dev)
    c.append(k.to(dev), v.to(dev), rope={"mode": 2})
    c.evict(keep, 0, torch.rand((2, 2, T), device=dev))
    for n in (1, 20):
        k2 = randn((2, 2, n, D), 62 + n, torch.float16)
        at = c.position()
        c.append(k2.to(dev), k2.to(dev), rope={"mode": 2})
        assert c.position() == at + n
        turned = F.rope(k2.to(dev), torch.arange(at, at + n, device=dev), mode=2)
        one = g.KVCache(2, 2, 64, D, torch.float32 if kind in ref.TOP else kind, dev)
        one.append(turned, turned)
        got = c.read()[0][:, :, -n:]
        want = one.read()[0]
        if kind in ref.TOP:
            held = c.lengths[0] // 32 * 32  # what is quantized since has lost bits: compare the tail
            n_tail = min(n, c.lengths[0] - held)
            got, want = got[:, :, n - n_tail:], want[:, :, n - n_tail:]
        assert torch.equal(got, want)
    c.clear(0)
    assert c.position(0) == 0 and c.position(1) == T + 21
    c.append(k[:, :, :5].to(dev), v[:, :, :5].to(dev), rope={"mode": 2})
    turned = F.rope(k[:, :, :5].to(dev), torch.arange(5, device=dev), mode=2)
    one = g.KVCache(2, 2, 8, D, torch.float32 if kind in ref.TOP else kind, dev)
    one.append(turned, turned)
    assert torch.equal(c.read()[0][0, :, :5], one.read()[0][0, :, :5])


def test_a_session(dev):
    """Multi-axis keys into an 8-bit cache, a window that counts weights, an eviction, decode steps: against the
    same steps in float64."""
    B, H, Hkv, S, D, keep, recent, sec = 1, 8, 2, 210, 128, 96, 16, (24, 20, 20)
    pos = torch.randint(0, 4000, (3, B, S + 6))
    k, v, q = (randn((B, n, S + 6, D), 70 + n, torch.float16) for n in (Hkv, Hkv, H))
    qt = F.rope_axes(q.to(dev), pos.to(dev), sec).cpu()
    kt = F.rope_axes(k.to(dev), pos.to(dev), sec).cpu()
    c = g.KVCache(B, Hkv, S + 6, D, torch.int8, dev, block_tokens=64)
    c.append(k[:, :, :S].to(dev), v[:, :, :S].to(dev), rope={"positions": pos[..., :S].to(dev), "sections": sec})
    c.attention(qt[:, :, S - 12:S].to(dev), accumulate=0.0)
    w = c.weights().cpu()
    kept = c.evict(keep, recent).cpu()
    K, V = ref.held(kt[0, :, :S], torch.int8, 64), ref.held(v[0, :, :S], torch.int8, 64)
    rows = [torch.tensor(ref.chosen(w[0, h, :S], keep, recent)) for h in range(Hkv)]
    assert all(torch.equal(kept[0, h], rows[h]) for h in range(Hkv))
    K, V = (ref.held(torch.stack([x[h, rows[h]] for h in range(Hkv)]), torch.int8, 64) for x in (K, V))
    for i in range(S, S + 6):
        c.append(k[:, :, i:i + 1].to(dev), v[:, :, i:i + 1].to(dev), pos_offset=i, rope={"positions": pos[..., i:i + 1].to(dev), "sections": sec})
        K, V = torch.cat([K, kt[0, :, i:i + 1].double()], 1), torch.cat([V, v[0, :, i:i + 1].double()], 1)
        got = c.attention(qt[:, :, i:i + 1].to(dev))[0].double().cpu()
        out, mass, slack, _, _ = ref.attend(qt[0, :, i:i + 1], ref.held(K, torch.int8, 64), ref.held(V, torch.int8, 64))
        assert ((got - out).abs() <= ref.bounds(out, mass, slack, keep + 6, torch.float16)).all(), i


def test_other_stream(dev):
    k = randn((1, 2, 300, 64), 80, torch.float16).to(dev)
    q, w = randn((1, 4, 1, 64), 81, torch.float16).to(dev), torch.rand((1, 2, 300), device=dev)

    def run():
        c = g.KVCache(1, 2, 300, 64, torch.int8, dev)
        c.append(k, k)
        c.attention(q, accumulate=1.0)
        sums = c.weights().clone()
        kept = c.evict(100, 10, w)
        return [sums, kept, *c.read(), c.attention(q)]

    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", CACHES)
def test_memory_of_an_eviction_on_another_stream_is_not_given_away(dev, kind):
    """What a cache of one stream held is read by an eviction that waits on another, while the first goes on."""
    k, v = randn((2, 2, 500, 64), 90, torch.float16), randn((2, 2, 500, 64), 91, torch.float16)
    w = torch.rand(2, 2, 500, generator=torch.Generator().manual_seed(92))
    plain = make(dev, k, v, kind)
    plain.evict(100, 10, w.to(dev))
    want = plain.read()
    side = torch.cuda.Stream(dev)
    c, wd, other = make(dev, k, v, kind), w.to(dev), [torch.randn(2, 2, 500, 64, device=dev, dtype=torch.float16) for _ in range(2)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # (some milliseconds)
        c.evict(100, 10, wd)
    later = [g.KVCache(2, 2, 500, 64, kind, dev) for _ in range(3)]
    for x in later:
        x.append(*other)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(c.read(), want))


@pytest.mark.parametrize("kind", CACHES)
def test_many_rows_over_few_tokens_of_a_large_cache(dev, kind):
    """Sums from several column splits, whose parts take the room of the tokens held, not of the capacity."""
    k, v, q = (randn((1, 2, 90, 64), 93 + i, torch.float16) for i in range(3))
    q = randn((1, 32, 90, 64), 96, torch.float16)
    c = make(dev, k, v, kind, cap=200_000)
    c.attention(q.to(dev), accumulate=1.0)
    weight_checks(c, c.weights()[..., :1000], q, torch.zeros((1, 2, 90), dtype=torch.float64), 0.0, True, "large")
    assert c.weights()[..., 90:].abs().max().item() == 0.0


@pytest.mark.parametrize("kind", CACHES)
def test_nothing_to_evict_and_a_full_cache(dev, kind):
    k, v = randn((1, 2, 96, 64), 97, torch.float16), randn((1, 2, 96, 64), 98, torch.float16)
    c = make(dev, k[:, :, :70], v[:, :, :70], kind, cap=96)
    before = c.read()
    kept = c.evict(96, 0, torch.rand(1, 2, 70, device=dev))
    assert kept.tolist() == [[list(range(70)) + [-1] * 26] * 2] and c.lengths == [70] and c.position() == 70
    assert all(torch.equal(a, b) for a, b in zip(c.read(), before))
    c.append(k[:, :, 70:].to(dev), v[:, :, 70:].to(dev))  # to the last token of the capacity
    whole = make(dev, k, v, kind)
    assert all(torch.equal(a, b) for a, b in zip(c.read(), whole.read()))
    q = randn((1, 4, 1, 64), 99, torch.float16).to(dev)
    assert torch.equal(c.attention(q), whole.attention(q))
    with pytest.raises(RuntimeError, match="do not fit"):
        c.append(k[:, :, :1].to(dev), v[:, :, :1].to(dev))
    assert c.evict(1, 1, torch.rand(1, 2, 96, device=dev)).tolist() == [[[95], [95]]] and c.lengths == [1] and c.position() == 96
    assert torch.equal(c.read()[0][:, :, 0].half().cpu(), whole.read()[0][:, :, 95].half().cpu())


def test_refusals(dev):
    c = g.KVCache(1, 2, 50, 64, torch.int8, dev)
    k = torch.ones((1, 2, 40, 64), device=dev)
    c.append(k, k)
    w = torch.ones((1, 2, 40), device=dev)
    for keep, recent in ((0, 0), (51, 0), (10, 11), (10, -1), (-5, 0)):
        with pytest.raises(RuntimeError, match="keep must be in"):
            c.evict(keep, recent, w)
    for bad in (w[..., :39], w[:, :1], w[0], w[..., None]):
        with pytest.raises(RuntimeError, match="weights must be"):
            c.evict(10, 0, bad)
    with pytest.raises(RuntimeError, match="must be a float tensor"):
        c.evict(10, 0, w.long())
    with pytest.raises(RuntimeError, match="must be in \\[0, 1\\]"):
        c.attention(torch.ones((1, 4, 1, 64), device=dev), accumulate=1.5)
    with pytest.raises(RuntimeError, match="at least one row"):
        c.attention(torch.ones((1, 4, 0, 64), device=dev), accumulate=1.0)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        c.attention(torch.ones((1, 4, 1, 64), device=dev, dtype=torch.float64), accumulate=1.0)
    with pytest.raises(RuntimeError, match="fewer than"):
        c.attention(torch.ones((1, 4, 41, 64), device=dev), accumulate=1.0)
    assert c.lengths == [40] and c.position() == 40
    wide = g.KVCache(1, 1, 8, 300, torch.float32, dev)
    wide.append(torch.ones((1, 1, 2, 300), device=dev), torch.ones((1, 1, 2, 300), device=dev))
    with pytest.raises(RuntimeError, match="head_dim must be at most 256"):
        wide.attention(torch.ones((1, 1, 1, 300), device=dev), accumulate=1.0)
