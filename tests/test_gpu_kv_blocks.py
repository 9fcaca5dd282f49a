"""The 8-bit block cache on the GPU: the values it stands for, bit for bit, however the tokens came; attention
over them by the kernels that read the codes and by those that read the values first, against float64."""

import math

import pytest
import torch

import gguf_train_amd as g
from gguf_train_amd import _C
from gguf_train_amd.nn import functional as F

import _kv_ref as ref
from _util import randn

pytestmark = pytest.mark.gpu

KINDS = [torch.int8, torch.float8_e4m3fn]


def cache_of(dev, k, v, kind, block, cap=None, pieces=None):
    B, Hkv, T, D = k.shape
    c = g.KVCache(B, Hkv, cap or max(T, 1), D, kind, dev, block_tokens=block)
    at = 0
    for n in pieces or [T]:
        c.append(k[:, :, at:at + n].to(dev), v[:, :, at:at + n].to(dev))
        at += n
    assert at == T
    return c


def held_equal(c, k, v, kind, block):
    for got, x in zip(c.read(), (k, v)):
        want = ref.held(x, kind, block)
        got = got.double().cpu()
        assert got.shape == want.shape
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("dtype,B,Hkv,T,D", [
    (torch.float16, 2, 2, 300, 128), (torch.bfloat16, 1, 3, 257, 64), (torch.float32, 2, 1, 128, 80), (torch.float32, 1, 1, 1, 64),
    (torch.float16, 1, 2, 127, 256), (torch.bfloat16, 1, 1, 65, 1), (torch.float32, 1, 2, 130, 50), (torch.float64, 1, 1, 70, 130)])
def test_values(dev, kind, block, dtype, B, Hkv, T, D):
    k, v = randn((B, Hkv, T, D), 1, dtype, 3.0), randn((B, Hkv, T, D), 2, dtype, 0.01)
    if dtype == torch.float64:  # held as float32
        k, v = k.float().double(), v.float().double()
    held_equal(cache_of(dev, k, v, kind, block), k, v, kind, block)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [32, 128])
def test_values_do_not_depend_on_the_pieces(dev, kind, block):
    B, Hkv, T, D = 2, 2, 301, 64
    k, v = randn((B, Hkv, T, D), 3, torch.float16), randn((B, Hkv, T, D), 4, torch.float16)
    for pieces in ([1] * 301, [31, 1, 1, 31, 64, 128, 45], [128, 128, 45], [5, 290, 6], [300, 1]):
        held_equal(cache_of(dev, k, v, kind, block, pieces=pieces), k, v, kind, block)


@pytest.mark.parametrize("kind", KINDS)
def test_every_code_and_every_tie(dev, kind):
    """One block per scale: all codes, halfway points and their neighbours."""
    top = ref.TOP[kind]
    y = torch.linspace(-top, top, 32 * 64 - 2, dtype=torch.float64).float()
    if kind == torch.int8:
        halves = torch.arange(-127, 127).float() + 0.5
    else:
        codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
        halves = torch.cat([(codes[1:] + codes[:-1]) / 2, -(codes[1:] + codes[:-1]) / 2, codes])
    y[:len(halves)] = halves
    y[1000:1000 + len(halves)] = torch.nextafter(halves, torch.full_like(halves, 1e9))
    x = torch.cat([torch.tensor([top, -top]), y]).reshape(1, 1, 32, 64)
    for scale in (1.0, 2.0 ** -20, 2.0 ** 60):
        held_equal(cache_of(dev, x * scale, -x * scale, kind, 32), x * scale, -x * scale, kind, 32)


@pytest.mark.parametrize("kind", KINDS)
def test_zeros_extremes_infinities_and_nan(dev, kind):
    B, Hkv, T, D = 1, 2, 32 * 7 + 3, 64
    k, v = randn((B, Hkv, T, D), 5), randn((B, Hkv, T, D), 6)
    k[:, :, :32] = 0.0
    k[:, :, 32:64] *= 1e-42   # subnormal
    k[:, :, 64:96] *= 1e38
    v[0, 0, 100, 3] = math.inf
    v[0, 1, 130, 4] = math.nan
    k[0, 1, 165, 5] = -math.inf
    k[:, :, 192:224] = torch.tensor(3.0e38)
    held_equal(cache_of(dev, k, v, kind, 32), k, v, kind, 32)


@pytest.mark.parametrize("kind", KINDS)
def test_half_precision_reads(dev, kind):
    k, v = randn((1, 2, 100, 64), 7, torch.bfloat16), randn((1, 2, 100, 64), 8, torch.bfloat16)
    c = cache_of(dev, k, v, kind, 32)
    for dtype in (torch.float16, torch.bfloat16):  # both exact: the codes have at most 8 bits
        for a, b in zip(c.read(dtype), c.read()):
            assert a.dtype == dtype and torch.equal(a.float(), b)
    big = torch.full((1, 1, 32, 64), 65504.0, dtype=torch.float16)
    c = cache_of(dev, big, big, kind, 32)
    assert c.read()[0].max().item() == 65536.0 and c.read(torch.float16)[0].max().item() == 65504.0


def test_other_dtypes_of_cache_are_read_too(dev):
    k, v = randn((2, 2, 40, 64), 9), randn((2, 2, 40, 64), 10)
    for dtype in (torch.float32, torch.float16, torch.bfloat16, "q8_0"):
        c = g.KVCache(2, 2, 64, 64, dtype, dev)
        c.append(k.to(dev), v.to(dev))
        c.clear(1)
        c.append(k[:, :, :9].to(dev), v[:, :, :9].to(dev))
        rk, rv = c.read()
        assert tuple(rk.shape) == (2, 2, 49, 64) and rk[1, :, 9:].abs().max().item() == 0.0
        for got, store in ((rk, c.keys()), (rv, c.values())):
            dense = g.dequantize(store) if dtype == "q8_0" else store.float()
            assert torch.equal(got[0], dense[0, :, :49]) and torch.equal(got[1, :, :9], dense[1, :, :9])


@pytest.mark.parametrize("kind", KINDS)
def test_strided_mixed_and_host_rows(dev, kind):
    B, Hkv, T, D = 2, 3, 70, 64
    k, v = randn((B, Hkv, T, D), 11, torch.float16), randn((B, Hkv, T, D), 12, torch.float16)
    want = cache_of(dev, k, v, kind, 32).read()
    kd, vd = k.to(dev), v.to(dev)
    rows = [(kd.transpose(1, 2).contiguous().transpose(1, 2), vd), (torch.stack([kd, kd], -1)[..., 1], vd),
            (torch.cat([kd.new_zeros(1), kd.reshape(-1)])[1:].reshape(kd.shape), vd), (k, vd), (k, v), (kd.float(), vd),
            (kd.double(), v)]
    for a, b in rows:
        c = g.KVCache(B, Hkv, T, D, kind, dev)
        c.append(a, b)
        assert all(torch.equal(x, y) for x, y in zip(c.read(), want))


def test_q8_0_rows(dev):
    k, v = randn((1, 2, 40, 64), 13), randn((1, 2, 40, 64), 14)
    qk, qv = g.quantize(k.to(dev)), g.quantize(v.to(dev))
    c = g.KVCache(1, 2, 40, 64, torch.int8, dev)
    c.append(qk, qv)
    held_equal(c, g.dequantize(qk).cpu(), g.dequantize(qv).cpu(), torch.int8, 32)


@pytest.mark.parametrize("kind", KINDS)
def test_rope_on_the_way_in(dev, kind):
    B, Hkv, T, D = 2, 2, 75, 64
    k, v = randn((B, Hkv, T, D), 15, torch.bfloat16), randn((B, Hkv, T, D), 16, torch.bfloat16)
    c = g.KVCache(B, Hkv, T, D, kind, dev)
    for a, b in ((0, 40), (40, 41), (41, 75)):
        c.append(k[:, :, a:b].to(dev), v[:, :, a:b].to(dev), pos_offset=a, rope={"mode": 2})
    turned = F.rope(k.to(dev), torch.arange(T, device=dev), mode=2).cpu()
    held_equal(c, turned, v, kind, 32)
    pos = torch.randint(0, 5000, (3, B, T))
    for dtype in (kind, torch.float16, "q8_0"):
        c = g.KVCache(B, Hkv, T, D, dtype, dev)
        for a, b in ((0, 40), (40, 41), (41, 75)):
            c.append(k[:, :, a:b].to(dev), v[:, :, a:b].to(dev), rope={"positions": pos[..., a:b].to(dev), "sections": (12, 10, 10)})
        plain = g.KVCache(B, Hkv, T, D, dtype, dev)
        plain.append(F.rope_axes(k.to(dev), pos.to(dev), (12, 10, 10)), v.to(dev))
        assert all(torch.equal(x, y) for x, y in zip(c.read(), plain.read()))


def attention_checks(c, q, k, v, kind, block, lengths, causal=True, scale=None, what=""):
    """Every sequence's rows against float64 over the values held, within the derived bound."""
    dev = c.device
    got = c.attention(q.to(dev), scale=scale, is_causal=causal)
    assert got.dtype == q.dtype and got.shape == q.shape
    got = got.double().cpu()
    for b, n in enumerate(lengths):
        out, mass, slack, _, _ = ref.attend(q[b], ref.held(k[b, :, :n], kind, block), ref.held(v[b, :, :n], kind, block), causal, scale)
        off, bound = (got[b] - out).abs(), ref.bounds(out, mass, slack, n, q.dtype)  # (a bound of 0: a row that sees one value of 0)
        assert (off <= bound).all(), (what, b, (off - bound).max().item())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,L,T,D,block", [
    (1, 1, 1, 1, 1, 64, 32), (1, 1, 1, 1, 31, 128, 32), (1, 4, 4, 1, 32, 64, 32), (2, 8, 2, 1, 33, 128, 32), (2, 8, 2, 1, 95, 80, 32),
    (1, 7, 1, 1, 777, 128, 64), (3, 16, 8, 1, 1000, 128, 128), (2, 4, 2, 1, 191, 256, 128), (1, 16, 1, 1, 300, 130, 32),
    (2, 8, 2, 5, 100, 128, 32), (1, 14, 2, 3, 640, 64, 64), (1, 4, 1, 16, 16, 128, 32), (1, 32, 1, 2, 500, 64, 128),
    (1, 8, 1, 13, 333, 128, 32), (1, 4, 1, 32, 70, 80, 32), (2, 3, 3, 20, 90, 200, 64), (1, 2, 2, 1, 5000, 64, 32),
    (1, 1, 1, 1, 40, 1, 32), (1, 2, 1, 2, 40, 50, 32)])
def test_attention_from_the_codes(dev, kind, dtype, B, H, Hkv, L, T, D, block):
    k, v, q = randn((B, Hkv, T, D), 20, dtype), randn((B, Hkv, T, D), 21, dtype), randn((B, H, L, D), 22, dtype)
    c = cache_of(dev, k, v, kind, block)
    attention_checks(c, q, k, v, kind, block, [T] * B, what="causal")
    assert "blocks of" in _C.last_launch()
    if L > 1:
        attention_checks(c, q, k, v, kind, block, [T] * B, causal=False, what="all")
    attention_checks(c, q, k, v, kind, block, [T] * B, scale=0.31, what="scale")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [32, 64, 128])
def test_an_append_to_the_end_of_the_room_leaves_its_neighbours_alone(dev, kind, block):
    """The grid is of the sequence that takes most blocks; the others are full before its last workgroup."""
    B, Hkv, D = 3, 2, 64
    c = g.KVCache(B, Hkv, 256, D, kind, dev, block_tokens=block)
    parts = [[randn((B, Hkv, n, D), 80 + n + i, torch.float16) for i in range(2)] for n in (99, 32, 125)]
    for i, (k, v) in enumerate(parts):
        c.append(k.to(dev), v.to(dev))
        if i == 0:
            c.clear(0)
    assert c.lengths == [157, 256, 256]
    for got, i in zip(c.read(), range(2)):
        whole, late = torch.cat([p[i] for p in parts], 2), torch.cat([p[i] for p in parts[1:]], 2)
        assert torch.equal(got[0, :, :157].double().cpu(), ref.held(late[0], kind, block))
        assert torch.equal(got[1:].double().cpu(), ref.held(whole[1:], kind, block))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ragged_sequences(dev, kind, dtype):
    B, H, Hkv, D = 3, 8, 2, 128
    c = g.KVCache(B, Hkv, 400, D, kind, dev)
    parts = [randn((B, Hkv, n, D), 30 + n, dtype) for n in (300, 300, 60, 60)]
    c.append(parts[0].to(dev), parts[1].to(dev))
    c.clear(1)
    c.append(parts[2].to(dev), parts[3].to(dev))
    assert c.lengths == [360, 60, 360] and [c.position(b) for b in range(B)] == [360, 60, 360]
    k, v = torch.cat([parts[0], parts[2]], 2), torch.cat([parts[1], parts[3]], 2)
    k[1, :, :60], v[1, :, :60] = parts[2][1], parts[3][1]
    for L in (1, 3):
        attention_checks(c, randn((B, H, L, D), 40 + L, dtype), k, v, kind, 32, c.lengths, what=f"L={L}")
    rk, _ = c.read()
    assert tuple(rk.shape) == (B, Hkv, 360, D) and rk[1, :, 60:].abs().max().item() == 0.0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,L,T,D,block", [
    (1, 8, 2, 200, 200, 128, 32), (1, 8, 2, 129, 500, 64, 64), (2, 3, 1, 190, 201, 80, 128), (1, 2, 1, 150, 150, 256, 32),
    (1, 1, 1, 700, 1000, 128, 32), (1, 4, 4, 65, 65, 64, 32)])
def test_prompts_from_the_codes(dev, kind, dtype, B, H, Hkv, L, T, D, block):
    """Rows that end at different units, over a cache of their own tokens or more."""
    k, v, q = randn((B, Hkv, T, D), 50, dtype), randn((B, Hkv, T, D), 51, dtype), randn((B, H, L, D), 52, dtype)
    c = cache_of(dev, k, v, kind, block)
    attention_checks(c, q, k, v, kind, block, [T] * B, what="causal")
    assert "blocks of" in _C.last_launch()
    attention_checks(c, q, k, v, kind, block, [T] * B, causal=False, what="all")


@pytest.mark.parametrize("kind", KINDS)
def test_ragged_prompts_from_the_codes(dev, kind):
    B, H, Hkv, D = 2, 4, 2, 64
    for dtype in (torch.float16, torch.float32):
        a, b = [randn((B, Hkv, 300, D), 53 + i, dtype) for i in range(2)], [randn((B, Hkv, 150, D), 55 + i, dtype) for i in range(2)]
        c = g.KVCache(B, Hkv, 500, D, kind, dev)
        c.append(a[0].to(dev), a[1].to(dev))
        c.clear(1)
        c.append(b[0].to(dev), b[1].to(dev))
        k, v = torch.cat([a[0], b[0]], 2), torch.cat([a[1], b[1]], 2)
        k[1, :, :150], v[1, :, :150] = b[0][1], b[1][1]
        attention_checks(c, randn((B, H, 150, D), 57, dtype), k, v, kind, 32, [450, 150])
        assert "blocks of" in _C.last_launch()


@pytest.mark.parametrize("kind", KINDS)
def test_prompts_that_fill_the_gpu(dev, kind):
    """float16 and bfloat16 rows for which the values are read first, against float64."""
    from _util import assert_close
    B, H, Hkv, T, D = 1, 32, 8, 260, 64
    for dtype in (torch.float16, torch.bfloat16):
        k, v, q = randn((B, Hkv, T, D), 50, dtype), randn((B, Hkv, T, D), 51, dtype), randn((B, H, T, D), 52, dtype)
        c = cache_of(dev, k, v, kind, 32)
        got = c.attention(q.to(dev))
        assert "read block cache" in _C.last_launch()
        out, _, _, _, _ = ref.attend(q[0], ref.held(k[0], kind, 32), ref.held(v[0], kind, 32))
        assert_close(got[0], out.numpy(), dtype, "prompt")


@pytest.mark.parametrize("kind", KINDS)
def test_float64_and_mixed_queries(dev, kind):
    k, v = randn((1, 2, 90, 64), 60, torch.bfloat16), randn((1, 2, 90, 64), 61, torch.bfloat16)
    c = cache_of(dev, k, v, kind, 32)
    K, V = ref.held(k[0], kind, 32), ref.held(v[0], kind, 32)
    for L in (1, 4):
        q = randn((1, 4, L, 64), 62, torch.float64)
        out, _, _, _, _ = ref.attend(q[0], K, V)
        assert (c.attention(q.to(dev))[0].cpu() - out).abs().max().item() <= 1e-10
    for dtype in (torch.float16, torch.float32):  # over tokens that came as bfloat16
        for L in (1, 90):
            q = randn((1, 4, L, 64), 63, dtype)
            out, mass, slack, _, _ = ref.attend(q[0], K, V)
            got = c.attention(q.to(dev))[0].double().cpu()
            tol = ref.bounds(out, mass, slack, 90, dtype) if L == 1 else 2e-3 * out.abs().clamp(min=1.0)
            assert ((got - out).abs() <= tol).all()


@pytest.mark.parametrize("kind", KINDS)
def test_blocks_of_very_different_size(dev, kind):
    """Value blocks from 1e-20 to 1e20 in size, the large ones of little weight; a block of zeros."""
    B, H, Hkv, T, D = 1, 4, 1, 32 * 6 + 5, 64
    k, v, q = randn((B, Hkv, T, D), 70), randn((B, Hkv, T, D), 71), randn((B, H, 1, D), 72)
    for j, s in enumerate((1e-20, 1e20, 0.0, 1.0, 1e10, 1e-3)):
        v[:, :, 32 * j:32 * j + 32] *= s
    for dtype in (torch.float32, torch.bfloat16):
        attention_checks(cache_of(dev, k, v, kind, 32), q.to(dtype), k, v, kind, 32, [T], what="sizes")
    v[:, :, 32:64] = 0.0
    v[:, :, 128:160] = 0.0
    tiny = v * 1e-20
    attention_checks(cache_of(dev, k, tiny, kind, 32), q, k, tiny, kind, 32, [T], what="tiny beside zeros")
    wide = q * 1e-18
    attention_checks(cache_of(dev, k * 1e18, v, kind, 32), wide, k * 1e18, v, kind, 32, [T], what="tiny queries, large keys")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("at", [5, 70])  # in a whole block, in the tail
def test_nan_and_infinities_reach_only_rows_that_see_them(dev, kind, what, at):
    B, H, Hkv, T, D = 1, 4, 2, 72, 64
    k, v = randn((B, Hkv, T, D), 80), randn((B, Hkv, T, D), 81)
    for bad in (math.nan, math.inf):
        kk, vv = k.clone(), v.clone()
        (kk if what == "k" else vv)[0, 0, at, 7] = bad
        c = cache_of(dev, kk, vv, kind, 32)
        q = randn((B, H, 4, D), 82)
        got = c.attention(q.to(dev)).cpu()
        K, V = ref.held(k[0], kind, 32), ref.held(v[0], kind, 32)
        out, mass, slack, _, _ = ref.attend(q[0], K, V)
        tol = ref.bounds(out, mass, slack, T, torch.float32)
        assert ((got[0, 2:] - out[2:]).abs() <= tol[2:]).all()  # the other kv head
        for l in range(4):
            sees = at < 64 or at <= T - 4 + l
            row = got[0, :2, l]
            if sees:
                assert torch.isnan(row).any(), (bad, l)
            else:
                assert ((row - out[:2, l]).abs() <= tol[:2, l]).all(), (bad, l)


@pytest.mark.parametrize("kind", KINDS)
def test_what_a_cleared_cache_held_does_not_come_back(dev, kind):
    B, H, Hkv, T, D = 1, 4, 2, 100, 64
    c = cache_of(dev, torch.full((B, Hkv, T, D), math.nan), torch.full((B, Hkv, T, D), math.nan), kind, 32)
    c.clear()
    assert c.lengths == [0] and c.position() == 0
    k, v, q = randn((B, Hkv, 37, D), 90), randn((B, Hkv, 37, D), 91), randn((B, H, 2, D), 92)
    c.append(k.to(dev), v.to(dev))
    attention_checks(c, q, k, v, kind, 32, [37])
    held_equal(c, k, v, kind, 32)


def test_strided_and_misaligned_queries(dev):
    B, H, Hkv, L, T, D = 2, 4, 2, 3, 70, 64
    k, v = randn((B, Hkv, T, D), 95, torch.float16), randn((B, Hkv, T, D), 96, torch.float16)
    c = cache_of(dev, k, v, torch.int8, 32)
    q = randn((B, H, L, D), 97, torch.float16).to(dev)
    want = c.attention(q)
    for view in (q.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([q.new_zeros(1), q.reshape(-1)])[1:].reshape(q.shape),
                 torch.stack([q, q], -1)[..., 0], q.cpu()):
        assert torch.equal(c.attention(view).to(dev), want)


def test_other_stream_and_two_caches(dev):
    H, Hkv, T, D = 8, 2, 700, 128
    kv = [randn((1, Hkv, T, D), 100 + i, torch.float16).to(dev) for i in range(4)]
    q = randn((1, H, 1, D), 110, torch.float16).to(dev)
    caches = [g.KVCache(1, Hkv, T, D, kind, dev) for kind in KINDS]
    for i, c in enumerate(caches):
        c.append(kv[2 * i], kv[2 * i + 1])
    want = [c.attention(q) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = []
    for s, c in zip(streams, caches):
        with torch.cuda.stream(s):
            got.append([c.attention(q) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for xs, w in zip(got, want) for x in xs)


def test_refusals(dev):
    c = g.KVCache(2, 2, 40, 64, torch.int8, dev)
    row = torch.ones((2, 2, 1, 64), device=dev)
    with pytest.raises(RuntimeError, match="holds 0 tokens"):
        c.attention(torch.ones((2, 4, 1, 64), device=dev))
    with pytest.raises(RuntimeError, match="do not fit the cache"):
        c.append(row.expand(2, 2, 41, 64), row.expand(2, 2, 41, 64))
    with pytest.raises(RuntimeError, match="do not continue"):
        c.append(row, row, pos_offset=3)
    with pytest.raises(RuntimeError, match="does not match the cache"):
        c.append(row[..., :32], row[..., :32])
    with pytest.raises(RuntimeError, match="block cache holds codes"):
        c.keys()
    with pytest.raises(RuntimeError, match="block cache holds codes"):
        c.values()
    with pytest.raises(ValueError, match="unsupported dtype"):
        c.read(torch.float64)
    for bad in ({"positions": torch.zeros(3, 1)}, {"sections": (12, 10, 10)}, {"positions": torch.zeros(3, 1), "sections": (12, 10, 10), "base": 1}):
        with pytest.raises(TypeError):
            c.append(row, row, rope=bad)
    with pytest.raises(RuntimeError, match="pos must be of shape"):
        c.append(row, row, rope={"positions": torch.zeros(3, 3, 1), "sections": (12, 10, 10)})
    assert c.lengths == [0, 0]
    rk, rv = c.read()
    assert tuple(rk.shape) == (2, 2, 0, 64)
    assert tuple(c.attention(torch.ones((2, 4, 0, 64), device=dev)).shape) == (2, 4, 0, 64)
