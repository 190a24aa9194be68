"""Tree drafts over a KV cache in the model dtype or in 8 bits, against plain implementations in 64 bits:
metadata, quantising append and read-back, attention, acceptance, compaction, and a round of them together.

Tolerances.  Integers, masks, stored bytes and read-back values are exact.  Attention: with p the softmax
weights and A = sum p |v|,
  output rounding            u_out |ref|            u = eps / 2: bf16 2^-8, fp32 2^-24
  weights rounded for PV     u_p A                  bf16 cache 2^-8, 8-bit caches (f16 weights) 2^-11, fp32 none
  scores                     2 e_s A                e_s = 2^-24 (D + 8) max_j sum_d |q_d k_jd| / sqrt(D), fp32 sums
  exp, sums over the keys    2^-20 A                two ulp of the exponential, fp32 sums of split ranges
and f16 weights below 2^-14 of a row's largest are subnormal: 2^-25 max|v| per key on top.
"""

import ctypes as C
import math

import numpy as np
import pytest
import torch

from thesis_b200 import lib
from thesis_b200 import tree as tr
from thesis_b200.config import ModelConfig
from thesis_b200.model import build_rope_cache

pytestmark = pytest.mark.gpu

QMAX = {"e4m3": 448.0, "int8": 127.0}
BAD_INDEX = 1 << 3
FORMATS = ["bf16", "e4m3", "int8"]


# ----------------------------------------------------------------- plain implementations
def quantise(x, fmt):
    """(stored values as fp64, exponent bytes) by the definition, numpy fp64."""
    x = np.asarray(x, dtype=np.float64)
    top = np.abs(x).max(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(top > 0, np.ceil(np.log2(top / QMAX[fmt])), -100)
    e = np.where(np.isfinite(e), e, -100)
    e = np.where(top > QMAX[fmt] * 2.0 ** e, e + 1, e)                 # log2 may round either way at a border
    e = np.where(top <= QMAX[fmt] * 2.0 ** (e - 1), e - 1, e)
    e = np.maximum(e, -100)
    bad = ~np.isfinite(x).all(-1)
    u = np.where(bad[..., None], 0, x) / 2.0 ** e[..., None]
    if fmt == "int8":
        u = np.rint(u)
    else:
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(u), 2.0 ** -6))) - 3)
        u = np.rint(u / step) * step
    return u, np.where(bad, 255, e + 127).astype(np.uint8)


def ancestors(parents):
    T = len(parents)
    m = np.zeros((T, T), dtype=bool)
    for i in range(T):
        j = i
        while j >= 0:
            m[i, j] = True
            j = parents[j]
    return m


def depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def random_tree(T, rng):
    return [-1] + [int(rng.integers(max(0, i - 1 - i // 2), i)) for i in range(1, T)]


def values64(cache, layer=0):
    out = []
    for d, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
        x = d[layer].double()
        if e is not None:
            f = torch.exp2(e[layer].double() - 127)
            x = x * torch.where(e[layer] == 255, torch.full_like(f, math.nan), f)[..., None]
        out.append(x)
    return out


def attend64(q, cache, blocks, sees, n_heads, layer=0):
    """(ref, A, e_s, vmax) per output row and head, fp64; sees[b][i] bool over the block's nodes."""
    K, V = values64(cache, layer)
    D, Hkv = cache.head_dim, cache.n_kv_heads
    G = n_heads // Hkv
    n = q.shape[0]
    ref = torch.zeros(n, n_heads, D, dtype=torch.float64, device=q.device)
    A = torch.zeros_like(ref)
    es = torch.zeros(n, n_heads, 1, dtype=torch.float64, device=q.device)
    vm = torch.zeros_like(es)
    start = 0
    for (row, ctx, _), see in zip(blocks, sees):
        T = len(see)
        for h in range(n_heads):
            k, v = K[row, h // G, :ctx + T], V[row, h // G, :ctx + T]
            for i in range(T):
                use = torch.tensor([True] * ctx + [bool(x) for x in see[i]], device=q.device)
                if not use.any():
                    continue
                qq = q[start + i, h * D:(h + 1) * D].double()
                kk, vv = k[use], v[use]
                s = kk @ qq / math.sqrt(D)
                p = torch.softmax(s, 0)
                ref[start + i, h] = p @ vv
                A[start + i, h] = p @ vv.abs()
                es[start + i, h] = 2.0 ** -24 * (D + 8) * ((kk.abs() @ qq.abs()).max() / math.sqrt(D))
                vm[start + i, h] = vv.abs().max()
        start += T
    return ref, A, es, vm


def check_attention(out, q, cache, blocks, sees, n_heads, layer=0):
    ref, A, es, vm = attend64(q, cache, blocks, sees, n_heads, layer)
    got = out.view(ref.shape).double()
    u_out = 2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -24
    if out.dtype == torch.float32:
        u_p, sub = 0.0, 0.0
    else:
        u_p, sub = (2.0 ** -8, 0.0) if cache.format == "bf16" else (2.0 ** -11, 2.0 ** -25 * max(c + len(s) for (_, c, _), s in zip(blocks, sees)))
    tol = u_out * ref.abs() * (1 + 2.0 ** -7) + A * (u_p * (1 + 2.0 ** -7) + 2 * es + 2.0 ** -20) + sub * vm + 1e-30
    err = (got - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol).nan_to_num(math.inf).max()), torch.nonzero(bad)[:4].tolist())


# ----------------------------------------------------------------- set-up
def make_cache(dev, fmt, B, Hkv, S, D, layers=1, seed=0):
    """A cache with content everywhere (stands in for earlier calls and for stale slots)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    c = tr.KVCache(layers, B, Hkv, S, D, fmt, dev)
    for d, e in ((c.k, c.k_exp), (c.v, c.v_exp)):
        x = torch.randn(c.k.shape, device=dev, generator=g) * torch.exp(0.5 * torch.randn(*c.k.shape[:4], 1, device=dev, generator=g))
        if e is None:
            d.copy_(x)
        else:
            u, eb = quantise(x.bfloat16().double().cpu().numpy(), fmt)
            d.copy_(torch.from_numpy(u).float().to(d.dtype).to(dev) if fmt == "e4m3" else torch.from_numpy(u).to(torch.int8).to(dev))
            e.copy_(torch.from_numpy(eb).to(dev))
    return c


def queries(dev, n, width, seed=1, dtype=torch.bfloat16):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(n, width, device=dev, generator=g) * 1.5).to(dtype)


def sees_of(blocks):
    out = []
    for _, _, p in blocks:
        out.append(np.tril(np.ones((p, p), dtype=bool)) if isinstance(p, int) else ancestors(p))
    return out


def tables(dev, S, D):
    cfg = ModelConfig(vocab_size=8, dim=64, n_layers=1, n_heads=1, n_kv_heads=1, head_dim=D, intermediate_size=64, rope_theta=500000.0)
    cos, sin = build_rope_cache(cfg, S)
    return cos.to(dev).contiguous(), sin.to(dev).contiguous()


# ----------------------------------------------------------------- metadata
@pytest.mark.parametrize("T", [1, 2, 31, 64, 65, 200, 256])
def test_tree_meta(cuda_dev, T):
    rng = np.random.default_rng(T)
    cache = make_cache(cuda_dev, "int8", 3, 1, 512, 64)
    blocks = [(2, 5, random_tree(T, rng)), (0, 0, [-1]), (1, 200, random_tree(max(1, T // 2), rng)), (1, 17, max(1, T - 1))]
    t = tr.TreeBatch(blocks, cache)
    t.check()
    start = 0
    for (row, ctx, p), see in zip(blocks, sees_of(blocks)):
        n = len(see)
        d = depths(p) if not isinstance(p, int) else list(range(n))
        assert t.tok_pos[start:start + n].tolist() == [ctx + x for x in d]
        assert t.tok_slot[start:start + n].tolist() == list(range(ctx, ctx + n))
        assert t.tok_row[start:start + n].tolist() == [row] * n
        words = t.mask[start:start + n].cpu().numpy().view(np.uint64)
        bits = (words[:, np.arange(n) // 64] >> (np.arange(n) % 64).astype(np.uint64)) & np.uint64(1)
        assert (bits.astype(bool) == see).all()
        start += n


def test_tree_meta_reports_what_does_not_fit(cuda_dev):
    cache = make_cache(cuda_dev, "int8", 3, 1, 128, 64)
    for col, bad in ((0, -1), (0, 5), (1, 0), (1, 5), (2, 3), (2, -1), (3, -1), (3, 126)):
        t = tr.TreeBatch([(0, 3, [-1, 0]), (1, 7, [-1, 0, 0])], cache)
        t.check()
        t.blk[1, col] = bad
        t.update()
        with pytest.raises(lib.EesdError):
            t.check()
        t.check()                                                     # cleared
        assert t.tok_slot[:2].tolist() == [3, 4]
    t = tr.TreeBatch([(0, 3, [-1, 0, 1])], cache)
    t.parent[2] = 2
    t.update()
    with pytest.raises(lib.EesdError):
        t.check()
    assert t.tok_pos.tolist() == [3, 4, 3]


# ----------------------------------------------------------------- append and read-back
def rope64(x, cos, sin, dtype):
    """[n, h, D] in the model dtype's roundings; products of two bf16 or fp32 numbers are exact in fp64."""
    r = (lambda t: t.to(dtype).double())
    c, s = r(cos)[:, None], r(sin)[:, None]
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h].double(), x[..., h:].double()
    a = r(x1 * c[..., :h]) - r(x2 * s[..., :h])
    b = r(x2 * c[..., h:]) + r(x1 * s[..., h:])
    return r(torch.cat([a, b], -1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("fmt", ["model", "e4m3", "int8"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (4, 1, 128), (3, 3, 128), (10, 2, 64)])
def test_append_and_read_back(cuda_dev, dtype, fmt, H, Hkv, D):
    fmt = ("bf16" if dtype == torch.bfloat16 else "f32") if fmt == "model" else fmt
    rng = np.random.default_rng(H + D)
    cache = make_cache(cuda_dev, fmt, 4, Hkv, 192, D, layers=2, seed=3)
    before = [t.view(torch.uint8).clone() if t.dtype.itemsize == 1 else t.clone()
              for t in (cache.k, cache.v, cache.k_exp, cache.v_exp) if t is not None]
    blocks = [(3, 100, random_tree(9, rng)), (0, 0, random_tree(13, rng)), (1, 127, 65), (2, 63, 1)]
    t = tr.TreeBatch(blocks, cache)
    n = t.n_tokens
    width = (H + 2 * Hkv) * D
    wide = queries(cuda_dev, n, width + 24, seed=H, dtype=dtype)
    wide[5, H * D:] = 0                                               # K and V of zeros
    wide[6] *= 1e-20
    wide[7] *= 1e20
    wide[8, H * D + 3] = math.inf                                     # one K head with an infinity
    wide[9, (H + 2 * Hkv) * D - 1] = math.nan                         # one V head with a NaN
    qkv = wide[:, :width]                                             # strided rows
    keep = wide.clone()
    cos, sin = tables(cuda_dev, 192, D)
    q_out = torch.full((n, H * D), 7.0, dtype=dtype, device=cuda_dev)
    tr.kv_append(qkv, cache, t, cos, sin, q_out=q_out, layer=1)
    t.check()
    assert torch.equal(wide.view(torch.uint8), keep.view(torch.uint8))
    x = qkv.reshape(n, H + 2 * Hkv, D)
    pos = t.tok_pos.long()
    turned = rope64(x[:, :H + Hkv], cos[pos], sin[pos], dtype)
    wantq, k, v = turned[:, :H], turned[:, H:], x[:, H + Hkv:].double()
    assert torch.equal(q_out.double().view(n, H, D).nan_to_num(123), wantq.nan_to_num(123))
    row, slot = t.tok_row.long(), t.tok_slot.long()
    ko, vo = (torch.empty(n, Hkv, D, dtype=dtype, device=cuda_dev) for _ in range(2))
    tr.kv_read(cache, t.tok_row, t.tok_slot, ko, vo, layer=1, status=t.status)
    t.check()
    for want, data, exps, got in ((k, cache.k, cache.k_exp, ko), (v, cache.v, cache.v_exp, vo)):
        if exps is None:
            assert torch.equal(data[1][row, :, slot].double().nan_to_num(123), want.nan_to_num(123))
            assert torch.equal(got.double().nan_to_num(123), want.nan_to_num(123))
            continue
        u, e = quantise(want.cpu().numpy(), fmt)
        assert (exps[1][row, :, slot].cpu().numpy() == e).all()
        raw = data.view(torch.uint8)[1][row, :, slot].view(data.dtype)
        assert (raw.double().cpu().numpy() == u).all()
        val = np.where((e == 255)[..., None], np.nan, u * 2.0 ** (e.astype(np.float64) - 127)[..., None])
        assert np.array_equal(got.double().cpu().numpy(), val, equal_nan=True)
        fin = np.isfinite(want.cpu().numpy()).all(-1)
        assert fin.sum() == fin.size - 1
    # everything else is as it was: the other layer, other rows, slots before and behind
    now = [c.view(torch.uint8).clone() if c.dtype.itemsize == 1 else c.clone()
           for c in (cache.k, cache.v, cache.k_exp, cache.v_exp) if c is not None]
    for a, b in zip(before, now):
        assert torch.equal(a[0], b[0])
        b[1][row, :, slot] = a[1][row, :, slot]
        assert torch.equal(a, b)
    # in place: the same rotated q
    tr.kv_append(qkv, cache, t, cos, sin, layer=1)
    assert torch.equal(wide[:, :H * D].contiguous().view(torch.uint8), q_out.view(torch.uint8))
    assert torch.equal(wide[:, H * D:].contiguous().view(torch.uint8), keep[:, H * D:].contiguous().view(torch.uint8))


def test_append_matches_the_unquantised_append(cuda_dev):
    """Model-dtype cache, a chain: bit-identical to eesd_rope_kv_append."""
    H, Hkv, D, S = 8, 2, 128, 128
    a, b = (make_cache(cuda_dev, "bf16", 2, Hkv, S, D) for _ in range(2))
    t = tr.TreeBatch([(1, 60, 9), (0, 0, 5)], a)
    qkv = queries(cuda_dev, t.n_tokens, (H + 2 * Hkv) * D)
    cos, sin = tables(cuda_dev, S, D)
    old = qkv.clone()
    lib.call("eesd_rope_kv_append", lib.BF16, old.data_ptr(), t.tok_pos.data_ptr(), t.tok_row.data_ptr(), t.n_tokens, H, Hkv, D,
             cos.data_ptr(), sin.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), 2, S, None, lib.stream_ptr())
    tr.kv_append(qkv, a, t, cos, sin)
    assert torch.equal(qkv, old) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_append_rotates_every_bf16_as_the_unquantised_append(cuda_dev):
    """The same with random bit patterns: subnormals, the largest values, infinities (NaN compared as NaN)."""
    H, Hkv, D, S = 8, 2, 64, 256
    a, b = (tr.KVCache(1, 1, Hkv, S, D, "bf16", cuda_dev) for _ in range(2))
    t = tr.TreeBatch([(0, 0, 256)], a)
    rng = np.random.default_rng(3)
    bits = rng.integers(0, 1 << 16, (256, (H + 2 * Hkv) * D)).astype(np.uint16)
    bits[64:128] &= 0x83ff                                              # at most 2^-119, half of them subnormal in products
    bits[128:192] = bits[128:192] & 0x80ff | 0x7e80                     # at least 2^126: sums that overflow
    qkv = torch.from_numpy(bits.view(np.int16)).to(cuda_dev).view(torch.bfloat16)
    cos, sin = tables(cuda_dev, S, D)
    old = qkv.clone()
    lib.call("eesd_rope_kv_append", lib.BF16, old.data_ptr(), t.tok_pos.data_ptr(), t.tok_row.data_ptr(), t.n_tokens, H, Hkv, D,
             cos.data_ptr(), sin.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), 1, S, None, lib.stream_ptr())
    tr.kv_append(qkv, a, t, cos, sin)
    for x, w in ((qkv, old), (a.k, b.k), (a.v, b.v)):
        same = (x.contiguous().view(torch.int16) == w.contiguous().view(torch.int16)) | (x.isnan() & w.isnan())
        assert same.all(), int((~same).sum())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_exponent_borders(cuda_dev, fmt):
    """Largest values on both sides of every border Q 2^e, halfway values, the clamp at 2^-100."""
    D, Q = 64, QMAX[fmt]
    cache = make_cache(cuda_dev, fmt, 1, 1, 1024, D)
    tops = []
    for e in (-101, -100, -99, -20, -1, 0, 1, 5, 100, 119, 120, 121, 122):
        for m in (Q, Q * (1 + 2.0 ** -7), Q * (1 - 2.0 ** -8), Q / 2, 1.0):
            if m * 2.0 ** e < 3e38:
                tops.append(m * 2.0 ** e)
    top = torch.tensor(tops, dtype=torch.float64).float().bfloat16().to(cuda_dev)
    n = len(tops)
    g = torch.Generator(device=cuda_dev).manual_seed(0)
    frac = torch.randint(-256, 257, (n, D), device=cuda_dev, generator=g).float() / 256
    x = (frac * top[:, None].float()).bfloat16()
    x[:, 17] = top
    t = tr.TreeBatch([(0, 0, n)], cache)
    qkv = torch.cat([torch.zeros(n, D, device=cuda_dev).bfloat16(), x, -x], 1)
    cos = torch.ones(1024, D, device=cuda_dev)
    tr.kv_append(qkv, cache, t, cos, torch.zeros_like(cos))
    for data, exps, want in ((cache.k, cache.k_exp, x), (cache.v, cache.v_exp, -x)):
        u, e = quantise(want.double().cpu().numpy(), fmt)
        assert (exps[0, 0, 0, :n].cpu().numpy() == e).all()
        assert (data.view(torch.uint8)[0, 0, 0, :n].view(data.dtype).double().cpu().numpy() == u).all()


def test_append_and_read_skip_what_is_out_of_range(cuda_dev):
    cache = make_cache(cuda_dev, "int8", 2, 1, 64, 64)
    t = tr.TreeBatch([(0, 10, 4)], cache)
    t.check()
    qkv = queries(cuda_dev, 4, 3 * 64)
    cos, sin = tables(cuda_dev, 64, 64)
    k0 = cache.k.clone()
    for name, bad in (("tok_pos", 64), ("tok_pos", -1), ("tok_slot", 64), ("tok_slot", -1), ("tok_row", 2), ("tok_row", -1)):
        v = getattr(t, name)
        old = int(v[2])
        v[2] = bad
        cache.k.copy_(k0)
        q = torch.full((4, 64), 5.0, dtype=torch.bfloat16, device=cuda_dev)
        tr.kv_append(qkv, cache, t, cos, sin, q_out=q)
        with pytest.raises(lib.EesdError):
            t.check()
        assert (q[2] == 5).all() and (q[3] != 5).any()
        assert torch.equal(cache.k[0, 0, 0, 12], k0[0, 0, 0, 12]) and not torch.equal(cache.k[0, 0, 0, 13], k0[0, 0, 0, 13])
        if name != "tok_pos":
            ko = torch.full((4, 1, 64), 5.0, dtype=torch.bfloat16, device=cuda_dev)
            tr.kv_read(cache, t.tok_row, t.tok_slot, ko, None, status=t.status)
            with pytest.raises(lib.EesdError):
                t.check()
            assert (ko[2] == 5).all() and (ko[1] != 5).any()
        v[2] = old


# ----------------------------------------------------------------- attention
SHAPES = [(4, 2, 64), (8, 1, 128), (32, 8, 128), (3, 3, 64), (10, 2, 128), (6, 2, 64)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_attention_trees(cuda_dev, fmt, H, Hkv, D):
    rng = np.random.default_rng(H * D)
    cache = make_cache(cuda_dev, fmt, 6, Hkv, 448, D, seed=H)
    blocks = [(0, 0, [-1]), (5, 1, random_tree(2, rng)), (1, 63, random_tree(5, rng)), (2, 120, random_tree(31, rng)),
              (4, 383, random_tree(64, rng)), (3, 254, random_tree(3, rng))]
    t = tr.TreeBatch(blocks, cache)
    wide = queries(cuda_dev, t.n_tokens, (H + 2 * Hkv) * D, seed=D)
    q = wide[:, :H * D]
    out = tr.tree_attention(q, cache, t)
    t.check()
    check_attention(out, q, cache, blocks, sees_of(blocks), H)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,T", [(0, 1), (0, 2), (15, 1), (16, 1), (63, 1), (64, 1), (65, 1), (127, 2), (128, 17), (0, 130), (77, 200)])
def test_attention_causal(cuda_dev, fmt, D, ctx, T):
    cache = make_cache(cuda_dev, fmt, 2, 2, 320, D, seed=ctx)
    blocks = [(1, ctx, T), (0, 3, 1)]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, 8 * D, seed=T)
    out = tr.tree_attention(q, cache, t)
    t.check()
    check_attention(out, q, cache, blocks, sees_of(blocks), 8)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 9, 40, 150])
def test_attention_long_context(cuda_dev, fmt, T):
    """The key range is split over CTAs; a fixed split gives the same bits alone and in a batch."""
    H, Hkv, D, ctx = 8, 2, 128, 9000
    rng = np.random.default_rng(T)
    cache = make_cache(cuda_dev, fmt, 2, Hkv, 9216, D, seed=T)
    p = random_tree(T, rng)
    blocks = [(1, ctx, p), (0, 300, p[:max(1, T // 2)])]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, H * D)
    some = sorted({0, T // 3, T - 1})
    out = tr.tree_attention(q, cache, t)
    t.check()
    sees = sees_of(blocks)
    one = [(1, ctx, p)]
    # a few nodes of the long block, checked one by one
    for i in some:
        K, V = values64(cache)
        use = torch.tensor([True] * ctx + [bool(x) for x in sees[0][i]], device=q.device)
        for h in (0, H - 1):
            kk, vv = K[1, h // (H // Hkv), :ctx + T][use], V[1, h // (H // Hkv), :ctx + T][use]
            qq = q[i, h * D:(h + 1) * D].double()
            s = kk @ qq / math.sqrt(D)
            w = torch.softmax(s, 0)
            want, a = w @ vv, w @ vv.abs()
            u_p, sub = (2.0 ** -8, 0) if fmt == "bf16" else (2.0 ** -11, 2.0 ** -25 * (ctx + T))
            e_s = 2.0 ** -24 * (D + 8) * (kk.abs() @ qq.abs()).max() / math.sqrt(D)
            tol = (2.0 ** -8 * want.abs() + u_p * a) * (1 + 2.0 ** -7) + a * (2 * e_s + 2.0 ** -20) + sub * vv.abs().max()
            assert ((out[i, h * D:(h + 1) * D].double() - want).abs() <= tol).all()
    fixed = tr.tree_attention(q, cache, t, split_keys=512)
    alone = tr.TreeBatch(one, cache)
    o1 = tr.tree_attention(q[:T], cache, alone, split_keys=512)
    assert torch.equal(o1, fixed[:T])


@pytest.mark.parametrize("fmt", ["f32", "e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_fp32(cuda_dev, fmt, D):
    rng = np.random.default_rng(D)
    cache = make_cache(cuda_dev, fmt, 3, 2, 256, D)
    blocks = [(2, 100, random_tree(20, rng)), (0, 0, random_tree(3, rng)), (1, 31, random_tree(33, rng))]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, 6 * D, dtype=torch.float32)
    out = tr.tree_attention(q, cache, t)
    t.check()
    check_attention(out, q, cache, blocks, sees_of(blocks), 6)


@pytest.mark.parametrize("fmt", ["f32"] + FORMATS)
@pytest.mark.parametrize("T,G", [(6, 2), (24, 4)])
def test_attention_masked_places_do_not_reach_a_node(cuda_dev, fmt, T, G):
    """An arbitrary mask with empty rows; NaN and infinities in slots that nobody sees, and in slots that only
    some nodes see: the others' outputs are as if the values were finite; a node that sees one gets it."""
    Hkv, D, ctx = 2, 64, 37
    H = G * Hkv
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    rng = np.random.default_rng(5)
    cache = make_cache(cuda_dev, fmt, 2, Hkv, 192, D)
    see = rng.random((T, T)) < 0.4                                     # not even causal
    see[2] = False
    blocks = [(1, ctx, [-1] * T), (0, 0, [-1] * T)]
    t = tr.TreeBatch(blocks, cache)
    t.mask.copy_(torch.from_numpy(np.tile((see * (1 << np.arange(T, dtype=np.int64))).sum(1).reshape(T, 1), (2, 1))))
    q = queries(cuda_dev, t.n_tokens, H * D, dtype=dt)
    clean = tr.tree_attention(q, cache, t)
    check_attention(clean, q, cache, blocks, [see, see], H)
    assert (clean[T + 2] == 0).all()                                   # no context and an empty row
    # slots behind the block, and rows of nobody
    poison = 3
    for row, c in ((1, ctx), (0, 0)):
        for slot, kind in ((c + T, math.nan), (c + T + 1, math.inf), (c + T + 9, -math.inf), (c + poison, math.nan)):
            if cache.quantised:
                cache.k_exp[0, row, :, slot] = 255
                cache.v_exp[0, row, :, slot] = 255
            else:
                cache.k[0, row, :, slot] = kind
                cache.v[0, row, :, slot, ::3] = kind
    out = tr.tree_attention(q, cache, t)
    t.check()
    blind = torch.from_numpy(np.tile(~see[:, poison], 2))
    assert torch.equal(out[blind], clean[blind])
    got = out[~blind].view(-1, H, D)[:, :, ::3]
    assert torch.isnan(got).all()


def test_attention_infinite_value_of_a_seen_slot(cuda_dev):
    """V = +-inf in one element of a slot that some nodes see: they get that infinity, the others nothing."""
    for T, ctx in ((6, 20), (40, 100)):
        cache = make_cache(cuda_dev, "bf16", 1, 2, 192, 64)
        rng = np.random.default_rng(T)
        p = random_tree(T, rng)
        see = ancestors(p)
        t = tr.TreeBatch([(0, ctx, p)], cache)
        q = queries(cuda_dev, T, 8 * 64)
        clean = tr.tree_attention(q, cache, t)
        cache.v[0, 0, :, ctx + 1, 5] = math.inf
        cache.v[0, 0, :, ctx + 2, 7] = -math.inf
        out = tr.tree_attention(q, cache, t)
        o, c = out.view(T, 8, 64), clean.view(T, 8, 64)
        for i in range(T):
            w = c[i].clone()
            if see[i, 1]:
                w[:, 5] = math.inf
            if see[i, 2]:
                w[:, 7] = -math.inf
            same = torch.ones(64, dtype=torch.bool, device=cuda_dev)
            same[[5, 7]] = False
            assert torch.equal(o[i][:, same], w[:, same])
            for d in (5, 7):
                if w[0, d].isinf():
                    assert torch.equal(o[i][:, d], w[:, d])
                else:
                    assert o[i][:, d].isfinite().all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_attention_extreme_scales(cuda_dev, fmt):
    """Scores far apart, keys and values of very different size: nothing overflows on the way."""
    H, Hkv, D, ctx, T = 8, 2, 128, 333, 12
    rng = np.random.default_rng(0)
    cache = make_cache(cuda_dev, fmt, 1, Hkv, 384, D)
    if cache.quantised:
        cache.k_exp[0, 0, :, 10:20] += 20
        cache.k_exp[0, 0, :, 30:60] -= 60
        cache.v_exp[0, 0, 0, 100:110] += 90
        cache.v_exp[0, 0, 1, :] -= 25
        cache.v_exp[0, 0, 1, 0] += 20
    else:
        cache.k[0, 0, :, 10:20] *= 2.0 ** 20
        cache.k[0, 0, :, 30:60] *= 2.0 ** -60
        cache.v[0, 0, 0, 100:110] *= 2.0 ** 90
    p = random_tree(T, rng)
    t = tr.TreeBatch([(0, ctx, p)], cache)
    q = queries(cuda_dev, T, H * D)
    q[0] *= 2.0 ** -70
    q[1] *= 2.0 ** 60
    out = tr.tree_attention(q, cache, t)
    t.check()
    assert out.isfinite().all()
    ref, A, _, _ = attend64(q, cache, [(0, ctx, p)], [ancestors(p)], H)
    # scores of 1e6 in fp32 sums leave a row either one-hot or close to it: compare where the 64-bit row is
    # not near a tie, with the weights' rounding alone
    K, _ = values64(cache)
    got = out.view(T, H, D).double()
    u_p = 2.0 ** -8 if fmt == "bf16" else 2.0 ** -11
    for i in (0, 2, 5):
        for h in (0, H - 1):
            s = (K[0, h // 4, :ctx] @ q[i, h * D:(h + 1) * D].double() / math.sqrt(D)).sort(descending=True).values
            if s[0] - s[1] > 60 or s[0].abs() < 1e3:
                tol = 2.0 ** -7 * ref[i, h].abs() + 2 * u_p * A[i, h] + (2.0 ** -25 * ctx * A[i, h].max() if fmt != "bf16" else 0)
                assert ((got[i, h] - ref[i, h]).abs() <= tol * 1.1 + 1e-30).all(), (i, h)


def test_attention_leaves_other_rows(cuda_dev):
    """A block that does not fit is skipped and reported; its rows and the others' are as they were or right."""
    cache = make_cache(cuda_dev, "e4m3", 2, 2, 128, 64)
    blocks = [(0, 20, [-1, 0, 0]), (1, 50, [-1, 0, 1, 1])]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, 7, 4 * 64)
    good = tr.tree_attention(q, cache, t)
    for col, bad in ((0, -1), (0, 4), (1, 0), (1, 9), (2, 2), (3, 126), (3, -3)):
        t = tr.TreeBatch(blocks, cache)
        t.blk[1, col] = bad
        out = torch.full_like(good, 3.0)
        tr.tree_attention(q, cache, t, out)
        with pytest.raises(lib.EesdError):
            t.check()
        assert torch.equal(out[:3], good[:3]) and (out[3:] == 3).all()


def test_attention_is_repeatable_and_capturable(cuda_dev):
    """Same bits twice, on another stream, and from two replayed graphs that share a workspace in turn."""
    cache = make_cache(cuda_dev, "int8", 2, 2, 4224, 128)
    rng = np.random.default_rng(1)
    t = tr.TreeBatch([(0, 4100, random_tree(40, rng)), (1, 900, random_tree(7, rng))], cache)
    q = queries(cuda_dev, t.n_tokens, 8 * 128)
    q2 = queries(cuda_dev, t.n_tokens, 8 * 128, seed=9)
    ws = tr.attention_workspace(t, cache, 8)
    a = tr.tree_attention(q, cache, t, workspace=ws)
    b = tr.tree_attention(q2, cache, t, workspace=ws)
    assert torch.equal(a, tr.tree_attention(q, cache, t))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = [torch.zeros_like(a), torch.zeros_like(a)]
    graphs = []
    with torch.cuda.stream(s):
        for x, o in zip((q, q2), outs):
            tr.tree_attention(x, cache, t, o, workspace=ws)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                tr.tree_attention(x, cache, t, o, workspace=ws)
            graphs.append(g)
    torch.cuda.synchronize()
    for o in outs:
        o.zero_()
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], a) and torch.equal(outs[1], b)
    t.check()


def test_attention_matches_the_chain_attention(cuda_dev):
    """Chains over a bf16 cache: what eesd_attn_varlen_gqa computes, within the weights' rounding."""
    from thesis_b200.packing import pack

    H, Hkv, D, S = 32, 8, 128, 640
    cache = make_cache(cuda_dev, "bf16", 3, Hkv, S, D)
    blocks = [(0, 500, 5), (2, 63, 5), (1, 0, 5)]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, (H + 2 * Hkv) * D)
    new = tr.tree_attention(q[:, :H * D], cache, t)
    ph = pack(blocks, lib.load().eesd_attn_item_tokens(H, Hkv))
    parts = [torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32).reshape(-1)).to(cuda_dev)
             for a in (ph.tok_pos, ph.tok_row, ph.blk, ph.items)]
    b = lib.Batch(ph.n_tokens, ph.n_blocks, len(ph.items), ph.max_ctx, *(p.data_ptr() for p in parts))
    old = torch.zeros_like(new)
    lib.call("eesd_attn_varlen_gqa", lib.BF16, q.data_ptr(), H, Hkv, D, cache.k.data_ptr(), cache.v.data_ptr(), 3, S, b, 0, None, None,
             old.data_ptr(), None, lib.stream_ptr())
    _, A, _, _ = attend64(q[:, :H * D], cache, blocks, sees_of(blocks), H)
    err = (new.double() - old.double()).abs().view(A.shape)
    assert (err <= 2 * (2.0 ** -8 * A * 2) * 1.02).all()               # each side: weights and output rounded


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("H,Hkv,D,T", [(5, 1, 64, 256), (2, 2, 128, 256), (48, 1, 128, 1), (40, 1, 64, 3), (33, 1, 128, 9)])
def test_attention_widest_trees_and_groups(cuda_dev, fmt, H, Hkv, D, T):
    """The most nodes that a mask has, groups of more heads than a small tile has rows, and row counts that end in
    every part of the larger tiles."""
    rng = np.random.default_rng(T)
    cache = make_cache(cuda_dev, fmt, 3, Hkv, 576, D, seed=D)
    blocks = [(0, 190, random_tree(T, rng)), (2, 0, random_tree(max(1, T - 100), rng)), (1, 320, random_tree(T, rng))]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, H * D, seed=H)
    out = tr.tree_attention(q, cache, t)
    t.check()
    check_attention(out, q, cache, blocks, sees_of(blocks), H)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
@pytest.mark.parametrize("n", [1, 3, 60])
def test_attention_many_small_units(cuda_dev, fmt, n):
    """Ragged short contexts: runs that hold many units, or less than one, and CTAs that are left without a run."""
    H, Hkv, D = 16, 1, 64
    rng = np.random.default_rng(n)
    cache = make_cache(cuda_dev, fmt, 3, Hkv, 1088, D)
    for _ in range(4):
        blocks = [(int(rng.integers(3)), int(rng.choice([0, 1, 63, 64, 447, 449, 511, 513, 1000])), int(rng.integers(3, 25)))
                  for _ in range(n)]
        t = tr.TreeBatch(blocks, cache)
        q = queries(cuda_dev, t.n_tokens, H * D)
        out = tr.tree_attention(q, cache, t)
        t.check()
        check_attention(out, q, cache, blocks, sees_of(blocks), H)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("n", [30, 128, 129])
def test_attention_many_blocks(cuda_dev, fmt, n):
    """More CTAs than SMs with few rows each: the long blocks run first, every block once, equal lengths among them; one
    block does not fit and is skipped wherever it stands in that order."""
    H, Hkv, D = 12, 6, 64
    rng = np.random.default_rng(n)
    cache = make_cache(cuda_dev, fmt, 4, Hkv, 320, D)
    blocks = [(int(rng.integers(4)), int(rng.choice([0, 5, 5, 64, 200, 300])), int(rng.integers(1, 4))) for _ in range(n)]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, H * D)
    out = tr.tree_attention(q, cache, t)
    t.check()
    check_attention(out, q, cache, blocks, sees_of(blocks), H)
    t = tr.TreeBatch(blocks, cache)
    t.blk[n // 2, 3] = 2 ** 31 - 2                                     # T + ctx wraps
    start, T = int(t.blk[n // 2, 0]), int(t.blk[n // 2, 1])
    again = torch.full_like(out, 3.0)
    tr.tree_attention(q, cache, t, again)
    with pytest.raises(lib.EesdError):
        t.check()
    assert (again[start:start + T] == 3).all()
    again[start:start + T] = out[start:start + T]
    assert torch.equal(again, out)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("T", [3, 40])
def test_attention_reports_a_wait_that_runs_out(cuda_dev, fmt, T):
    """With a poll limit of 0 every pipeline wait gives up: the status word says so and the next call is right."""
    cache = make_cache(cuda_dev, fmt, 2, 2, 640, 128)
    rng = np.random.default_rng(T)
    blocks = [(0, 500, random_tree(T, rng)), (1, 64, random_tree(2, rng))]
    t = tr.TreeBatch(blocks, cache)
    q = queries(cuda_dev, t.n_tokens, 8 * 128)
    good = tr.tree_attention(q, cache, t)
    t.check()
    lib.call("eesd_set_option", lib.OPT_SPIN_LIMIT, 0)
    try:
        tr.tree_attention(q, cache, t)
        torch.cuda.synchronize()
    finally:
        lib.call("eesd_set_option", lib.OPT_SPIN_LIMIT, -1)
    with pytest.raises(lib.EesdError):
        t.check()
    assert torch.equal(tr.tree_attention(q, cache, t), good)
    t.check()


def test_attention_calls_at_once(cuda_dev):
    """Calls on two streams, each with its own workspace, while a third launches its round: the bits of calls one by one."""
    H, Hkv, D = 8, 2, 128
    rng = np.random.default_rng(5)
    caches = [make_cache(cuda_dev, f, 2, Hkv, 4352, D, seed=i) for i, f in enumerate(("e4m3", "bf16", "int8"))]
    trees = [tr.TreeBatch([(0, 4100, random_tree(T, rng)), (1, 700, random_tree(5, rng))], c) for T, c in zip((40, 60, 5), caches)]
    qs = [queries(cuda_dev, t.n_tokens, H * D, seed=i) for i, t in enumerate(trees)]
    want = [tr.tree_attention(q, c, t) for q, c, t in zip(qs, caches, trees)]
    ws = [tr.attention_workspace(t, c, H) for t, c in zip(trees, caches)]
    outs = [[torch.zeros_like(w) for _ in range(6)] for w in want]
    streams = [torch.cuda.Stream() for _ in trees]
    torch.cuda.synchronize()
    for k in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                tr.tree_attention(qs[i], caches[i], trees[i], outs[i][k], workspace=ws[i])
    torch.cuda.synchronize()
    for w, o, t in zip(want, outs, trees):
        t.check()
        assert all(torch.equal(w, x) for x in o)


def test_batch_and_cache_on_different_devices_are_refused(cuda_dev):
    cache = make_cache(cuda_dev, "e4m3", 1, 1, 64, 64)
    t = tr.TreeBatch([(0, 8, 2)], cache)
    cos, sin = tables(cuda_dev, 64, 64)
    q = queries(cuda_dev, 2, 64)
    t.device = torch.device("cuda", 7)
    with pytest.raises(ValueError):
        tr.tree_attention(q, cache, t)
    with pytest.raises(ValueError):
        tr.kv_append(queries(cuda_dev, 2, 3 * 64), cache, t, cos, sin)
    with pytest.raises(ValueError):
        tr.kv_compact(cache, t, torch.zeros(1, 2, dtype=torch.int32, device=cuda_dev), torch.ones(1, dtype=torch.int32, device=cuda_dev))


# ----------------------------------------------------------------- acceptance and compaction
def walk(y, ids, parents):
    path = [0]
    while True:
        kids = [j for j in range(len(parents)) if j > 0 and parents[j] == path[-1] and ids[j] == y[path[-1]]]
        if not kids:
            return path
        path.append(kids[0])


@pytest.mark.parametrize("fmt", ["f32"] + FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_accept_and_compact(cuda_dev, fmt, D):
    rng = np.random.default_rng(D)
    cache = make_cache(cuda_dev, fmt, 9, 2, 512, D, layers=3)
    trees = [[-1], random_tree(2, rng), random_tree(31, rng), random_tree(64, rng), random_tree(200, rng), random_tree(33, rng),
             list(range(-1, 255)), [-1] + [0] * 40]
    blocks = [(8 - i, 7 * i, p) for i, p in enumerate(trees)]
    t = tr.TreeBatch(blocks, cache)
    ids = rng.integers(0, 5, t.n_tokens).astype(np.int32)              # few tokens: ties between children
    y = rng.integers(0, 5, t.n_tokens).astype(np.int32)
    start = 0
    for k, p in enumerate(trees):
        for i in range(len(p)):
            kids = [j for j in range(len(p)) if p[j] == i]
            if kids and (k == 6 or rng.random() < 0.9):
                y[start + i] = ids[start + kids[int(rng.integers(len(kids)))]]
        start += len(p)
    yd, idd = torch.from_numpy(y).to(cuda_dev), torch.from_numpy(ids).to(cuda_dev)
    path = torch.full((len(trees), 256), 99, dtype=torch.int32, device=cuda_dev)
    n_acc, nxt = (torch.full((len(trees),), 99, dtype=torch.int32, device=cuda_dev) for _ in range(2))
    tr.tree_accept(yd, idd, t, path, n_acc, nxt)
    t.check()
    raw = [c.view(torch.uint8) if c.dtype.itemsize == 1 else c for c in (cache.k, cache.v, cache.k_exp, cache.v_exp) if c is not None]
    want = [c.clone() for c in raw]
    start = 0
    for b, (row, ctx, p) in enumerate(blocks):
        w = walk(y[start:start + len(p)], ids[start:start + len(p)], p)
        assert path[b].tolist() == w + [-1] * (256 - len(w))
        assert int(n_acc[b]) == len(w) - 1 and int(nxt[b]) == y[start + w[-1]]
        for c in want:
            c[:, row, :, ctx:ctx + len(w)] = c[:, row, :, [ctx + j for j in w]].clone()
        start += len(p)
    assert int(n_acc[6]) == 255
    tr.kv_compact(cache, t, path, n_acc)
    t.check()
    for a, b in zip(raw, want):
        assert torch.equal(a, b)


def test_accept_matches_greedy_accept_on_chains(cuda_dev):
    rng = np.random.default_rng(3)
    nv, T = 17, 6
    cache = make_cache(cuda_dev, "int8", nv, 1, 64, 64)
    t = tr.TreeBatch([(i, 2 * i, T) for i in range(nv)], cache)
    ids = rng.integers(0, 2, (nv, T)).astype(np.int32)
    y = torch.from_numpy(rng.integers(0, 2, nv * T).astype(np.int32)).to(cuda_dev)
    seq = torch.from_numpy(ids.copy()).to(cuda_dev)
    vinfo = torch.tensor([[i * T, T, i] for i in range(nv)], dtype=torch.int32, device=cuda_dev)
    acc = torch.zeros(nv, dtype=torch.int32, device=cuda_dev)
    lib.call("eesd_greedy_accept", y.data_ptr(), vinfo.data_ptr(), nv, seq.data_ptr(), T, acc.data_ptr(), lib.stream_ptr())
    path = torch.empty(nv, T, dtype=torch.int32, device=cuda_dev)
    n_acc, nxt = torch.empty_like(acc), torch.empty_like(acc)
    tr.tree_accept(y, torch.from_numpy(ids).to(cuda_dev).view(-1), t, path, n_acc, nxt)
    assert torch.equal(acc, n_acc) and torch.equal(nxt, seq[:, 0])


def test_accept_and_compact_report_what_does_not_fit(cuda_dev):
    cache = make_cache(cuda_dev, "int8", 2, 1, 64, 64)
    k0 = cache.k.clone()
    t = tr.TreeBatch([(0, 3, [-1, 0, 0, 1]), (1, 5, [-1, 0, 0])], cache)
    y = torch.zeros(7, dtype=torch.int32, device=cuda_dev)
    path = torch.empty(2, 4, dtype=torch.int32, device=cuda_dev)
    n_acc, nxt = (torch.empty(2, dtype=torch.int32, device=cuda_dev) for _ in range(2))
    t.blk[1, 1] = 9
    tr.tree_accept(y, y, t, path, n_acc, nxt)
    with pytest.raises(lib.EesdError):
        t.check()
    assert path[1].tolist() == [-1] * 4 and n_acc.tolist()[1] == -1 and nxt.tolist()[1] == -1 and path[0].tolist() == [0, 1, 3, -1]
    t.blk[1, 1] = 3
    for bad in ([0, 2, 2, -1], [0, 4, 5, -1], [0, 2, 1, -1], [-1, 0, 1, -1]):
        cache.k.copy_(k0)
        path[1] = torch.tensor(bad, device=cuda_dev)
        n_acc[1] = 2
        tr.kv_compact(cache, t, path, n_acc)
        with pytest.raises(lib.EesdError):
            t.check()
        assert torch.equal(cache.k[:, 1], k0[:, 1])
        assert torch.equal(cache.k[0, 0, 0, 5], k0[0, 0, 0, 6]) and torch.equal(cache.k[0, 0, 0, 4], k0[0, 0, 0, 4])
    for bad in (-1, 3, 100):
        n_acc[1] = bad
        tr.kv_compact(cache, t, path, n_acc)
        with pytest.raises(lib.EesdError):
            t.check()
        assert torch.equal(cache.k[:, 1], k0[:, 1])


# ----------------------------------------------------------------- a round of them together
@pytest.mark.parametrize("fmt", FORMATS)
def test_round_of_tree_drafts(cuda_dev, fmt):
    """Two layers, three rounds: append, attention, acceptance and compaction leave a cache that holds exactly the
    accepted tokens' keys and values at their positions, as a chain of those tokens appended at once would."""
    L, B, H, Hkv, D, S = 2, 3, 8, 2, 64, 256
    rng = np.random.default_rng(8)
    cos, sin = tables(cuda_dev, S, D)
    cache, plain = tr.KVCache(L, B, Hkv, S, D, fmt, cuda_dev), tr.KVCache(L, B, Hkv, S, D, fmt, cuda_dev)
    ctx = [0, 0, 0]
    history = [[[] for _ in range(B)] for _ in range(L)]              # accepted tokens' qkv rows
    for rnd in range(3):
        blocks = [(b, ctx[b], random_tree(int(rng.integers(3, 20)), rng)) for b in range(B)]
        t = tr.TreeBatch(blocks, cache)
        ws = tr.attention_workspace(t, cache, H)
        rows = []
        for layer in range(L):
            qkv = queries(cuda_dev, t.n_tokens, (H + 2 * Hkv) * D, seed=10 * rnd + layer)
            rows.append(qkv.clone())
            tr.kv_append(qkv, cache, t, cos, sin, layer=layer)
            out = tr.tree_attention(qkv[:, :H * D], cache, t, layer=layer, workspace=ws)
            check_attention(out, qkv[:, :H * D], cache, blocks, sees_of(blocks), H, layer)
        ids = torch.from_numpy(rng.integers(0, 2, t.n_tokens).astype(np.int32)).to(cuda_dev)
        y = torch.from_numpy(rng.integers(0, 2, t.n_tokens).astype(np.int32)).to(cuda_dev)
        path = torch.empty(B, t.max_nodes, dtype=torch.int32, device=cuda_dev)
        n_acc, nxt = (torch.empty(B, dtype=torch.int32, device=cuda_dev) for _ in range(2))
        tr.tree_accept(y, ids, t, path, n_acc, nxt)
        tr.kv_compact(cache, t, path, n_acc)
        t.check()
        for b in range(B):
            start, keep = int(t.blk[b, 0]), path[b, :int(n_acc[b]) + 1].tolist()
            for layer in range(L):
                history[layer][b] += [rows[layer][start + i] for i in keep]
            ctx[b] += len(keep)
    chain = tr.TreeBatch([(b, 0, ctx[b]) for b in range(B)], plain)
    for layer in range(L):
        tr.kv_append(torch.stack([r for b in range(B) for r in history[layer][b]]), plain, chain, cos, sin, layer=layer)
    for layer in range(L):
        for b in range(B):
            for x, w in ((cache.k, plain.k), (cache.v, plain.v), (cache.k_exp, plain.k_exp), (cache.v_exp, plain.v_exp)):
                if x is not None:
                    x, w = (z[layer, b, :, :ctx[b]] for z in (x, w))
                    assert torch.equal(x.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
def test_wrapped_tensors_are_the_cache(cuda_dev, fmt):
    """A cache over existing tensors, as a model's: written and read in place, the same bits as a cache of its own."""
    L, B, H, Hkv, D, S = 2, 2, 4, 2, 64, 128
    dt = torch.bfloat16 if fmt == "bf16" else torch.float32
    own = tr.KVCache(L, B, Hkv, S, D, fmt, cuda_dev)
    k, v = torch.zeros(L, B, Hkv, S, D, dtype=dt, device=cuda_dev), torch.zeros(L, B, Hkv, S, D, dtype=dt, device=cuda_dev)
    over = tr.KVCache.wrap(k, v)
    cos, sin = tables(cuda_dev, S, D)
    blocks = [(1, 0, 30), (0, 0, [-1, 0, 0, 2])]
    outs = []
    for cache in (own, over):
        t = tr.TreeBatch(blocks, cache)
        qkv = queries(cuda_dev, t.n_tokens, (H + 2 * Hkv) * D, dtype=dt)
        tr.kv_append(qkv, cache, t, cos, sin, layer=1)
        outs.append(tr.tree_attention(qkv[:, :H * D], cache, t, layer=1))
        t.check()
    assert torch.equal(*outs) and torch.equal(k, own.k) and torch.equal(v, own.v)
    assert k[1, 1, :, :30].abs().sum() > 0 and (k[0] == 0).all()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("T", [5, 40])
def test_cache_beyond_32_bit_offsets(cuda_dev, fmt, T):
    """The last row of a layer with more than 2^31 elements: the bits of the same round in a small cache."""
    H, Hkv, D, S, ctx = 4, 1, 128, 256, 200
    cos, sin = tables(cuda_dev, S, D)
    rng = np.random.default_rng(T)
    p = random_tree(T, rng)
    results = []
    for B in (2, 70000):
        cache = tr.KVCache(1, B, Hkv, S, D, fmt, cuda_dev)
        assert B == 2 or cache.k.numel() > 2 ** 31
        first = tr.TreeBatch([(B - 1, 0, ctx)], cache)
        tr.kv_append(queries(cuda_dev, ctx, (H + 2 * Hkv) * D, seed=1), cache, first, cos, sin)
        t = tr.TreeBatch([(B - 1, ctx, p)], cache)
        qkv = queries(cuda_dev, T, (H + 2 * Hkv) * D, seed=2)
        tr.kv_append(qkv, cache, t, cos, sin)
        out = tr.tree_attention(qkv[:, :H * D], cache, t)
        path = torch.tensor([[0, 2, 4] + [-1] * (T - 3)], dtype=torch.int32, device=cuda_dev)
        tr.kv_compact(cache, t, path, torch.tensor([2], dtype=torch.int32, device=cuda_dev))
        rows = torch.full((ctx + 3,), B - 1, dtype=torch.int32, device=cuda_dev)
        slots = torch.arange(ctx + 3, dtype=torch.int32, device=cuda_dev)
        k, v = (torch.zeros(ctx + 3, Hkv, D, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
        tr.kv_read(cache, rows, slots, k, v)
        first.check()
        t.check()
        results.append((out, k, v))
        del cache, first, t
        torch.cuda.empty_cache()
    assert all(torch.equal(a, b) for a, b in zip(*results)) and results[0][1][-1].abs().sum() > 0


def test_round_is_capturable(cuda_dev):
    """A whole round as one graph, replayed with other contents: the eager results."""
    L, B, H, Hkv, D, S = 2, 2, 4, 2, 64, 192
    cos, sin = tables(cuda_dev, S, D)
    cache = make_cache(cuda_dev, "e4m3", B, Hkv, S, D, layers=L)
    rng = np.random.default_rng(2)
    t = tr.TreeBatch([(0, 70, random_tree(12, rng)), (1, 3, random_tree(5, rng))], cache)
    n = t.n_tokens
    qkv = [queries(cuda_dev, n, (H + 2 * Hkv) * D, seed=i) for i in range(L)]
    q, out = torch.empty(n, H * D, dtype=torch.bfloat16, device=cuda_dev), [torch.empty(n, H * D, dtype=torch.bfloat16, device=cuda_dev) for _ in range(L)]
    ids, y = (torch.from_numpy(rng.integers(0, 2, n).astype(np.int32)).to(cuda_dev) for _ in range(2))
    path = torch.empty(B, t.max_nodes, dtype=torch.int32, device=cuda_dev)
    n_acc, nxt = (torch.empty(B, dtype=torch.int32, device=cuda_dev) for _ in range(2))
    ws = tr.attention_workspace(t, cache, H)

    def step():
        t.update()
        for i in range(L):
            tr.kv_append(qkv[i], cache, t, cos, sin, q_out=q, layer=i)
            tr.tree_attention(q, cache, t, out[i], layer=i, workspace=ws)
        tr.tree_accept(y, ids, t, path, n_acc, nxt)
        tr.kv_compact(cache, t, path, n_acc)

    state = [x.view(torch.uint8).clone() for x in (cache.k, cache.v, cache.k_exp, cache.v_exp)]

    def reset():
        for x, s in zip((cache.k, cache.v, cache.k_exp, cache.v_exp), state):
            x.view(torch.uint8).copy_(s)

    def result():
        torch.cuda.synchronize()
        return [o.clone() for o in out] + [path.clone(), n_acc.clone(), nxt.clone(), cache.k.view(torch.uint8).clone(), cache.v_exp.clone()]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    torch.cuda.synchronize()
    for seed in (5, 6):
        for i in range(L):
            qkv[i].copy_(queries(cuda_dev, n, (H + 2 * Hkv) * D, seed=seed + 10 * i))
        t.blk[0, 3] = 60 + seed
        y.copy_(torch.from_numpy(rng.integers(0, 2, n).astype(np.int32)))
        reset()
        step()
        want = result()
        reset()
        g.replay()
        for a, b in zip(result(), want):
            assert torch.equal(a, b)
    t.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("D", [64, 128])
def test_attention_one_row_tile_at_every_ring_position(cuda_dev, fmt, D):
    """33 to 128 query rows per KV head: two streams share the key tiles, at every number of tiles from 1 to 11 and one after
    another, so that a stage is reused at every distance and by either stream."""
    H, Hkv = 12, 1
    rng = np.random.default_rng(D)
    cache = make_cache(cuda_dev, fmt, 3, Hkv, 768, D, seed=D)
    for n in (4, 33):
        blocks = [(int(rng.integers(3)), 64 * int(rng.integers(11)) + int(rng.integers(50)), random_tree(int(rng.integers(3, 11)), rng))
                  for _ in range(n)]
        t = tr.TreeBatch(blocks, cache)
        q = queries(cuda_dev, t.n_tokens, H * D, seed=n)
        out = tr.tree_attention(q, cache, t)
        t.check()
        check_attention(out, q, cache, blocks, sees_of(blocks), H)
        fixed = tr.tree_attention(q, cache, t, split_keys=256)
        t.check()
        check_attention(fixed, q, cache, blocks, sees_of(blocks), H)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [3, 20, 60])
def test_attention_waits_that_run_out_part_of_the_way(cuda_dev, fmt, T):
    """Poll limits at which some roles give up while others have loads in flight: a call either reports it or is right, and
    what runs on the same SMs right behind it is right."""
    cache = make_cache(cuda_dev, fmt, 2, 2, 4224, 128)
    rng = np.random.default_rng(T)
    t = tr.TreeBatch([(0, 4100, random_tree(T, rng)), (1, 64, random_tree(2, rng))], cache)
    q = queries(cuda_dev, t.n_tokens, 8 * 128)
    ws, ws2 = (tr.attention_workspace(t, cache, 8) for _ in range(2))
    good = tr.tree_attention(q, cache, t, workspace=ws)
    t.check()
    outs = [torch.empty_like(good) for _ in range(2)]
    reported = 0
    try:
        for limit in (0, 1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, 128):
            for _ in range(3):
                lib.call("eesd_set_option", lib.OPT_SPIN_LIMIT, limit)
                tr.tree_attention(q, cache, t, outs[0], workspace=ws)
                lib.call("eesd_set_option", lib.OPT_SPIN_LIMIT, -1)
                tr.tree_attention(q, cache, t, outs[1], workspace=ws2)
                torch.cuda.synchronize()
                assert torch.equal(outs[1], good), limit
                try:
                    t.check()
                except lib.EesdError:
                    reported += 1
                else:
                    assert torch.equal(outs[0], good), limit
    finally:
        lib.call("eesd_set_option", lib.OPT_SPIN_LIMIT, -1)
    assert reported > 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ctx,p,H", [(9, 1, 8), (300, 1, 8), (63, 1, 8), (100, [-1, 0, 0, 1, 3], 8), (77, 20, 8), (100, "tree40", 8), (1000, 3, 8),
                                     (300, 1, 80), (64, 33, 80), (4400, 2, 8), (4400, 40, 8)], ids=str)
def test_attention_nonfinite_values_of_seen_slots(cuda_dev, D, ctx, p, H):
    """bf16 cache, K finite: NaN or an infinity in one element of V, in committed slots on both sides of every tile and
    group border and in the nodes' own: all nodes that see the slot get it, in that element alone; the others nothing."""
    Hkv = 2
    p = random_tree(40, np.random.default_rng(1)) if p == "tree40" else p
    T = p if isinstance(p, int) else len(p)
    see = sees_of([(0, ctx, p)])[0]
    cache = make_cache(cuda_dev, "bf16", 1, Hkv, 4480, D, seed=T)
    t = tr.TreeBatch([(0, ctx, p)], cache)
    q = queries(cuda_dev, T, H * D) * 0.25                              # no weight of a seen slot vanishes
    clean = {split: tr.tree_attention(q, cache, t, split_keys=split).view(T, H, D) for split in (0, 256)}
    slots = sorted({0, ctx - 1, ctx, ctx + T - 1, ctx // 16 * 16, ctx // 32 * 32, ctx // 64 * 64, max(0, ctx // 64 * 64 - 1)})
    for n, slot in enumerate(slots):
        value = (math.nan, math.inf, -math.inf)[n % 3]
        keep = cache.v[0, 0, :, slot, 5].clone()
        cache.v[0, 0, :, slot, 5] = value
        for split, want in clean.items():
            out = tr.tree_attention(q, cache, t, split_keys=split).view(T, H, D)
            t.check()
            for i in range(T):
                sees = slot < ctx or bool(see[i, slot - ctx])
                rest = torch.ones(D, dtype=torch.bool, device=cuda_dev)
                rest[5] = False
                assert torch.equal(out[i][:, rest], want[i][:, rest])
                got = out[i][:, 5]
                if not sees:
                    assert torch.equal(got, want[i][:, 5]), (slot, i)
                elif math.isnan(value):
                    assert got.isnan().all(), (slot, i)
                else:
                    assert (got == value).all(), (slot, i, got)
        cache.v[0, 0, :, slot, 5] = keep


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 40])
def test_attention_nan_in_a_range_of_vanishing_weight(cuda_dev, fmt, T):
    """A NaN of V in a slot whose weight is far below fp32, in another key range than the largest score: it is seen all the
    same (0 x NaN), whichever way the keys are split."""
    H, Hkv, D, ctx = 4, 1, 64, 1000
    cache = make_cache(cuda_dev, fmt, 1, Hkv, 1088, D)
    t = tr.TreeBatch([(0, ctx, T)], cache)
    q = queries(cuda_dev, T, H * D)
    q[:] = 1.0
    cache.k[0, 0, :, :ctx] = torch.zeros(1, device=cuda_dev).to(cache.k.dtype)
    cache.k[0, 0, :, 900] = torch.full((1,), 64.0, device=cuda_dev).to(cache.k.dtype)   # the score of 900: 512 2^e, all others' 0 or small
    if cache.quantised:
        cache.k_exp[0, 0, :, 900] = 127
        cache.v_exp[0, 0, :, 10] = 255
    else:
        cache.v[0, 0, :, 10] = math.nan
    for split in (0, 256, 512):
        out = tr.tree_attention(q, cache, t, split_keys=split)
        t.check()
        assert out.isnan().all(), split


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,H,Hkv,D", [(6, 8, 2, 64), (6, 8, 2, 128), (3, 2, 2, 128), (16, 4, 2, 64), (40, 8, 2, 128), (100, 4, 2, 64)])
def test_attention_large_keys_and_values_that_others_see(cuda_dev, fmt, T, H, Hkv, D):
    """Finite keys with scores far above the rest, and values of a far larger scale, in a slot that only some nodes see: not
    a bit of the others' rows changes."""
    ctx = 75
    rng = np.random.default_rng(T)
    p = random_tree(T, rng)
    see = ancestors(p)
    cache = make_cache(cuda_dev, fmt, 1, Hkv, 256, D, seed=T)
    t = tr.TreeBatch([(0, ctx, p)], cache)
    q = queries(cuda_dev, T, H * D)
    clean = tr.tree_attention(q, cache, t)
    for node in sorted({1, T // 2, T - 1}):
        blind = torch.from_numpy(~see[:, node])
        for part in ("k", "v"):
            x, e = getattr(cache, part), getattr(cache, part + "_exp")
            keep = (x if e is None else e)[0, 0, :, ctx + node].clone()
            for up in (3, 6, 40):
                if e is None:
                    x[0, 0, :, ctx + node] = keep * 2.0 ** up
                else:
                    e[0, 0, :, ctx + node] = keep + up
                out = tr.tree_attention(q, cache, t)
                t.check()
                assert torch.equal(out[blind], clean[blind]), (node, part, up)
                assert part == "k" and up == 3 or not torch.equal(out[~blind], clean[~blind])
            (x if e is None else e)[0, 0, :, ctx + node] = keep


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("T", [6, 40, 100])
def test_attention_largest_exponent_that_others_see(cuda_dev, fmt, T):
    """Values near the smallest scale, and one of the largest scale that a bf16 vector can have in a slot that only some
    nodes see: the others' rows keep every bit."""
    H, Hkv, D, ctx = 8, 2, 64, 75
    rng = np.random.default_rng(T)
    p = random_tree(T, rng)
    see = ancestors(p)
    cache = make_cache(cuda_dev, fmt, 1, Hkv, 256, D, seed=T)
    for down in (60, 90):
        cache.v_exp[:] = torch.clamp(cache.v_exp.int() - down, min=27).to(torch.uint8)
        t = tr.TreeBatch([(0, ctx, p)], cache)
        q = queries(cuda_dev, T, H * D)
        clean = tr.tree_attention(q, cache, t)
        check_attention(clean, q, cache, [(0, ctx, p)], [see], H)
        for node in (1, T - 1):
            keep = cache.v_exp[0, 0, :, ctx + node].clone()
            cache.v_exp[0, 0, :, ctx + node] = 247 if fmt == "int8" else 245
            out = tr.tree_attention(q, cache, t)
            t.check()
            blind = torch.from_numpy(~see[:, node])
            assert torch.equal(out[blind], clean[blind]), (down, node)
            cache.v_exp[0, 0, :, ctx + node] = keep


def check_weighted(out, q, cache, ctx, p, H, above, exact_keys=()):
    """As check_attention, for one block, with the f16 weights' subnormal step counted against what matters: their reference lies at
    most 2^above over the largest p_j max|v_j| of the row (not over the largest |v_j|), so a key loses at most
    2^-25 2^above of that.  ``exact_keys``: slots whose score has no rounding error."""
    K, V = values64(cache)
    T, D, G, see = len(p), cache.head_dim, H // cache.n_kv_heads, ancestors(p)
    got = out.view(T, H, D).double()
    for i in range(T):
        use = torch.tensor([True] * ctx + [bool(x) for x in see[i]], device=q.device)
        rough = use.clone()
        rough[list(exact_keys)] = False
        for h in range(H):
            k, v = K[0, h // G, :ctx + T], V[0, h // G, :ctx + T]
            qq = q[i, h * D:(h + 1) * D].double()
            w = torch.softmax(torch.where(use, k @ qq / math.sqrt(D), -math.inf), 0)
            ref, A = w @ v, w @ v.abs()
            es = 2.0 ** -24 * (D + 8) * (k[rough].abs() @ qq.abs()).max() / math.sqrt(D)
            sub = int(use.sum()) * 2.0 ** (above - 25) * (w * v.abs().amax(1)).max()
            tol = 2.0 ** -8 * ref.abs() * (1 + 2.0 ** -7) + A * (2.0 ** -11 * (1 + 2.0 ** -7) + 2 * es + 2.0 ** -20) + sub + 1e-30
            err = (got[i, h] - ref).abs()
            assert (err <= tol).all(), (i, h, float((err / tol).max()))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6, 40, 100])
def test_attention_large_values_of_small_weight(cuda_dev, fmt, D, T):
    """8-bit caches: a seen slot whose values are 2^20 to 2^70 times the others' and whose weight is far smaller still, or about
    the inverse of that: what the others contribute stays."""
    H, Hkv, ctx = 8, 2, 333
    p = random_tree(T, np.random.default_rng(T))
    q = 1.5 + 0.1 * queries(cuda_dev, T, H * D).float()
    q = q.bfloat16()
    for slot in (0, 50, ctx - 1):
        cache = make_cache(cuda_dev, fmt, 1, Hkv, 448, D, seed=D)
        cache.k[0, 0, :, slot] = torch.full((1,), -QMAX[fmt], device=cuda_dev).to(cache.k.dtype)
        cache.k_exp[0, 0, :, slot] = 127 + (-7 if fmt == "e4m3" else -5)     # -3.5, -4 each: scores of -42 to -68, weights of 2^-60 to 2^-98
        v0 = cache.v_exp[0, 0, :, slot].clone()
        for up in (20, 30, 50, 70):
            cache.v_exp[0, 0, :, slot] = v0 + up
            t = tr.TreeBatch([(0, ctx, p)], cache)
            out = tr.tree_attention(q, cache, t)
            t.check()
            check_weighted(out, q, cache, ctx, p, H, 1 if T * H // Hkv <= 32 else 9)   # tcgen05: a tile's largest scale stands for all of its keys within 2^8


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 6, 40, 100])
def test_attention_keys_of_scales_far_apart(cuda_dev, fmt, D, T):
    """8-bit caches: a key 2^10 to 2^60 times the others that q is orthogonal to: its score is 0, and the others' keep their bits."""
    H, Hkv, ctx = 8, 2, 333
    p = random_tree(T, np.random.default_rng(T))
    q = torch.ones(T, H * D, dtype=torch.bfloat16, device=cuda_dev)
    for slot in (0, 50, 200, ctx - 1):
        cache = make_cache(cuda_dev, fmt, 1, Hkv, 448, D, seed=D)
        sign = torch.where(torch.arange(D, device=cuda_dev) % 2 == 0, 1.0, -1.0)
        cache.k[0, 0, :, slot] = (sign * QMAX[fmt]).to(cache.k.dtype)
        for up in (10, 20, 30, 60):
            cache.k_exp[0, 0, :, slot] = 120 + up
            t = tr.TreeBatch([(0, ctx, p)], cache)
            out = tr.tree_attention(q, cache, t)
            t.check()
            check_weighted(out, q, cache, ctx, p, H, 1 if T * H // Hkv <= 32 else 9, exact_keys=[slot])


@pytest.mark.parametrize("chains", [True, False])
def test_blocks_cut_short_leave_padding(cuda_dev, chains):
    """Blocks shortened or moved on the device: tokens that no block covers any more are no tokens.  They get slot -1, are
    neither written to the cache nor reported, and their rows of the outputs stay as they were."""
    H, Hkv, D, S = 4, 2, 64, 256
    cos, sin = tables(cuda_dev, S, D)
    rng = np.random.default_rng(4)
    sizes = [5, 4, 7, 3]
    blocks = [(b, 10 * b + 3, n if chains else random_tree(n, rng)) for b, n in enumerate(sizes)]
    first = [0, 5, 9, 16]
    cache = make_cache(cuda_dev, "int8", 4, Hkv, S, D)
    for edits, gone in (([(0, 1, 3)], [3, 4]), ([(3, 1, 1)], [17, 18]), ([(0, 0, 2), (0, 1, 3)], [0, 1]), ([(1, 1, 1), (2, 1, 2)], [6, 7, 8] + list(range(11, 16))),
                        ([(0, 1, 1), (1, 1, 1), (2, 1, 1), (3, 1, 1)], [i for i in range(19) if i not in first])):
        if not chains and edits[0][1] == 0:
            continue                                                    # a tree that starts elsewhere needs other parents
        t = tr.TreeBatch(blocks, cache, max_ctx=S)
        t.check()
        for b, col, v in edits:
            t.blk[b, col] = v
        t.blk[:, 3] += 2                                               # stale slots would lie under the new tokens
        t.update()
        t.check()
        live = torch.tensor([i not in gone for i in range(19)], device=cuda_dev)
        for x in (t.tok_slot, t.tok_row, t.tok_pos):
            assert (x[~live] == -1).all() and (x[live] >= 0).all()
        before = [x.view(torch.uint8).clone() for x in (cache.k, cache.v, cache.k_exp, cache.v_exp)]
        qkv = queries(cuda_dev, 19, (H + 2 * Hkv) * D)
        q = torch.full((19, H * D), 7.0, dtype=torch.bfloat16, device=cuda_dev)
        tr.kv_append(qkv, cache, t, cos, sin, q_out=q)
        k, out = torch.full((19, Hkv, D), 7.0, dtype=torch.bfloat16, device=cuda_dev), torch.full_like(q, 7.0)
        tr.kv_read(cache, t.tok_row, t.tok_slot, k, None, status=t.status)
        tr.tree_attention(q, cache, t, out)
        t.check()
        for x in (q, k, out):
            assert (x[~live] == 7).all() and (x[live] != 7).any()
        row, slot = t.tok_row[live].long(), t.tok_slot[live].long()
        for x, b in zip((cache.k, cache.v, cache.k_exp, cache.v_exp), before):
            x = x.view(torch.uint8).clone()
            x[0, row, :, slot] = b[0, row, :, slot]
            assert torch.equal(x, b)


def test_tokens_of_a_block_out_of_range_get_no_slot(cuda_dev):
    """A block whose place does not fit is reported, and the tokens that it leaves behind are not written."""
    cache = make_cache(cuda_dev, "int8", 3, 1, 128, 64)
    for col, bad in ((0, -1), (0, 50), (1, 0), (1, -3), (1, 50)):
        t = tr.TreeBatch([(0, 3, 2), (1, 7, 3), (2, 9, 4)], cache)
        t.check()
        t.blk[1, col] = bad
        t.update()
        with pytest.raises(lib.EesdError):
            t.check()
        assert t.tok_slot.tolist() == [3, 4, -1, -1, -1, 9, 10, 11, 12], (col, bad)
        t.blk[0, col], t.blk[2, col] = bad, bad
        t.update()
        with pytest.raises(lib.EesdError):
            t.check()
        assert t.tok_slot.tolist() == [-1] * 9


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_compact_refuses_blocks_that_share_slots(cuda_dev, fmt):
    """Two blocks of one row: where their slots overlap both are reported and left, as are no others; apart they are moved."""
    cache = make_cache(cuda_dev, fmt, 3, 2, 128, 64, layers=2)
    state = [x.view(torch.uint8).clone() for x in (cache.k, cache.v, cache.k_exp, cache.v_exp) if x is not None]
    raw = [x.view(torch.uint8) for x in (cache.k, cache.v, cache.k_exp, cache.v_exp) if x is not None]
    for second, shared in ((4, True), (7, True), (0, True), (8, False), (60, False)):
        for x, s in zip(raw, state):
            x.copy_(s)
        blocks = [(1, 4, 4), (1, second, 4 if second else 5), (2, 4, 4)]
        t = tr.TreeBatch(blocks, cache)
        t.check()
        path = torch.full((3, t.max_nodes), -1, dtype=torch.int32, device=cuda_dev)
        path[:, :3] = torch.tensor([0, 2, 3], device=cuda_dev)
        n_acc = torch.full((3,), 2, dtype=torch.int32, device=cuda_dev)
        tr.kv_compact(cache, t, path, n_acc)
        if shared:
            with pytest.raises(lib.EesdError):
                t.check()
        else:
            t.check()
        want = [s.clone() for s in state]
        for b, (row, ctx, _) in enumerate(blocks):
            if b == 2 or not shared:
                for w, s in zip(want, state):
                    w[:, row, :, ctx + 1:ctx + 3] = s[:, row, :, ctx + 2:ctx + 4]
        for x, w in zip(raw, want):
            assert torch.equal(x, w), second


def test_compact_over_many_blocks(cuda_dev):
    """More blocks than a CTA has threads, every one looked at for shared slots."""
    n = 600
    cache = make_cache(cuda_dev, "int8", n, 1, 64, 64)
    k = cache.k.clone()
    t = tr.TreeBatch([((7 * b) % n, 3 + b % 5, 4) for b in range(n)], cache)
    path = torch.tensor([[0, 2, 3, -1]] * n, dtype=torch.int32, device=cuda_dev)
    n_acc = torch.full((n,), 2, dtype=torch.int32, device=cuda_dev)
    tr.kv_compact(cache, t, path, n_acc)
    t.check()
    for b in (0, 255, 256, 511, 599):
        row, ctx = (7 * b) % n, 3 + b % 5
        assert torch.equal(cache.k[0, row, 0, ctx + 1:ctx + 3], k[0, row, 0, ctx + 2:ctx + 4])
    t.blk[590, 2], t.blk[590, 3] = t.blk[3, 2], t.blk[3, 3] + 3          # meets block 3
    cache.k.copy_(k)
    tr.kv_compact(cache, t, path, n_acc)
    with pytest.raises(lib.EesdError):
        t.check()
    assert torch.equal(cache.k[0, 21], k[0, 21]) and not torch.equal(cache.k[0, 28], k[0, 28])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T", [1, 40])
def test_attention_range(cuda_dev, fmt, T):
    """|q| up to 2^100: the rows come out as the value of their largest score (the next one is far below); over a bf16 cache |V| up
    to 2^100 as well, within the usual tolerance."""
    H, Hkv, D, ctx = 4, 1, 64, 400
    p = random_tree(T, np.random.default_rng(T))
    cache = make_cache(cuda_dev, fmt, 1, Hkv, 512, D, seed=T)
    t = tr.TreeBatch([(0, ctx, p)], cache)
    q = queries(cuda_dev, T, H * D)
    big = (q.float() * (2.0 ** 100 / float(q.float().abs().max()))).bfloat16()
    out = tr.tree_attention(big, cache, t).view(T, H, D).double()
    t.check()
    K, V = values64(cache)
    see = ancestors(p)
    checked = 0
    for i in range(T):
        use = torch.tensor([True] * ctx + [bool(x) for x in see[i]], device=cuda_dev)
        k, v = K[0, 0, :ctx + T][use], V[0, 0, :ctx + T][use]
        for h in range(H):
            qq = big[i, h * D:(h + 1) * D].double()
            s = k @ qq / math.sqrt(D)
            top = s.sort(descending=True)
            off = 2 * 2.0 ** -24 * (D + 8) * float((k.abs() @ qq.abs()).max()) / math.sqrt(D)   # of two scores, as they are summed
            assert out[i, h].isfinite().all()
            if top.values[0] - top.values[1] > off + 200:
                want = v[top.indices[0]]
                assert ((out[i, h] - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20)).all(), (i, h)
                checked += 1
    assert checked > T * H // 2
    if fmt == "bf16":
        cache.v *= 2.0 ** 100 / float(cache.v.float().abs().max())
        out = tr.tree_attention(q, cache, t)
        t.check()
        check_attention(out, q, cache, [(0, ctx, p)], [see], H)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("T", [6, 40, 100])
def test_attention_scales_that_others_see_leave_small_weights(cuda_dev, fmt, T):
    """8-bit caches: a row whose largest score has a value of small scale, zero in half of the dims, so that those dims are the sum of
    weights at the end of f16; values of a large scale that only other nodes see must not change how they are rounded."""
    H, Hkv, D, ctx = 8, 2, 64, 75
    p = random_tree(T, np.random.default_rng(T))
    see = ancestors(p)
    cache = make_cache(cuda_dev, fmt, 1, Hkv, 256, D, seed=T)
    cache.k[0, 0, :, 70] = torch.full((1,), QMAX[fmt], device=cuda_dev).to(cache.k.dtype)
    cache.k_exp[0, 0, :, 70] = 127 + (-9 if fmt == "e4m3" else -7)       # 0.88, 0.99 each: scores of about 11, 12
    cache.v_exp[0, 0, :, 70] -= 5
    cache.v.view(torch.uint8)[0, 0, :, 70, ::2] = 0
    t = tr.TreeBatch([(0, ctx, p)], cache)
    q = (1.5 + 0.1 * queries(cuda_dev, T, H * D).float()).bfloat16()
    clean = tr.tree_attention(q, cache, t)
    check_weighted(clean, q, cache, ctx, p, H, 1 if T * H // Hkv <= 32 else 9)
    for node in sorted({1, T // 2, T - 1}):
        keep = cache.v_exp[0, 0, :, ctx + node].clone()
        cache.v_exp[0, 0, :, ctx + node] = keep + 20
        out = tr.tree_attention(q, cache, t)
        t.check()
        blind = torch.from_numpy(~see[:, node])
        assert torch.equal(out[blind], clean[blind]), node
        cache.v_exp[0, 0, :, ctx + node] = keep
