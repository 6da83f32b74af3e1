"""linear, its packed weights and the adapters of many requests (GPU), against 64 bits.

A result is the f32 sum of the products rounded once to bf16. With S the sum of the
products' magnitudes, the f32 sums are off by at most 2 (K + R + 16) 2^-24 S (every
addition rounds by at most 2^-24 of a partial sum that S bounds; twice that for what the
matrix cores' own order may add), the adapters' inner values, carried in two bf16 above 64
tokens, by another 2^-16 of the adapters' share of S, and the rounding to bf16 by 2^-8."""

from __future__ import annotations

import ctypes
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


def _gen(dev, *seed):
    g = torch.Generator(device=dev)
    g.manual_seed(zlib.crc32(repr(seed).encode()))
    return g


def _randn(g, dev, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=dev) * std).to(torch.bfloat16)


def make(dev, T, K, N, weights="w8c", rows="bf16", seed=0):
    """x as ``linear`` takes it, the weight, and both in 64 bits."""
    from kappa_amd.qwen3 import Q8Rows, Q8Weight

    g = _gen(dev, T, K, N, weights, rows, seed)
    if rows == "q8":
        v = torch.randint(-127, 128, (T, K), generator=g, device=dev).to(torch.int8)
        s = torch.rand(T, 1, generator=g, device=dev) * 0.02 + 0.005
        x, xd = Q8Rows(v, s), v.double() * s.double()
    else:
        x = _randn(g, dev, T, K)
        xd = x.double()
    if weights == "bf16":
        w = _randn(g, dev, K, N, std=K**-0.5)
        return x, w, xd, w.double()
    q = torch.randint(-128, 128, (K, N), generator=g, device=dev).to(torch.int8)
    s = (torch.rand(1, N, generator=g, device=dev) + 0.5) * 0.01 * K**-0.5
    if weights == "w8t":
        s = s[0, 0].to(torch.bfloat16)
    return x, Q8Weight(q, s), xd, q.double() * s.double()


def make_adapters(dev, T, K, N, L, R, seed=0, none=True):
    g = _gen(dev, T, K, N, L, R, seed)
    a = _randn(g, dev, L, K, R, std=K**-0.5)
    b = _randn(g, dev, L, R, N, std=R**-0.5)
    f = torch.rand(L, generator=g, device=dev) * 2 - 0.5
    ad = torch.randint(-1 if none else 0, L, (T,), generator=g, device=dev).to(torch.int32)
    return a, b, f, ad


def check(y, xd, wd, K, lora=None, R=0):
    """y against xd @ wd with the adapters (a, b, factor, adapter)."""
    want, S = xd @ wd, xd.abs() @ wd.abs()
    slack = torch.zeros_like(S)
    if lora is not None:
        a, b, f, ad = lora
        for i in range(a.shape[0]):
            rows = torch.nonzero(ad == i).squeeze(1)
            if len(rows):
                A, B, fi = a[i].double(), b[i].double(), f[i].double()
                want[rows] += (xd[rows] @ A) @ B * fi
                part = (xd[rows].abs() @ A.abs()) @ B.abs() * fi.abs()
                S[rows] += part
                slack[rows] += part
    tol = 2 * (K + R + 16) * 2.0**-24 * S + 2.0**-16 * slack
    off = (y.double() - want).abs()
    bad = off > 2.0**-8 * (want.abs() + tol) + tol
    assert not bad.any(), (int(bad.sum()), float(off[bad].max()), torch.nonzero(bad)[:4].tolist())
    assert y.dtype == torch.bfloat16 and y.shape == want.shape


KINDS = [("bf16", "bf16"), ("w8c", "bf16"), ("w8t", "bf16"), ("w8c", "q8"), ("w8t", "q8")]
SIZES = [
    (1, 64, 16), (1, 2048, 512), (2, 128, 33), (7, 100, 31), (16, 192, 130), (17, 256, 64), (33, 1000, 257),
    (48, 512, 100), (64, 2048, 96), (65, 64, 1), (65, 128, 128), (127, 320, 130), (129, 1000, 257), (300, 512, 1000),
    (512, 1, 40), (700, 2048, 640),
]  # fmt: skip


@pytest.mark.parametrize("weights,rows", KINDS)
@pytest.mark.parametrize("T,K,N", SIZES)
def test_linear(dev, T, K, N, weights, rows):
    from kappa_amd.qwen3 import linear, prepack_linear

    x, w, xd, wd = make(dev, T, K, N, weights, rows)
    p = prepack_linear(w)
    y = linear(x, p)
    check(y, xd, wd, K)
    assert torch.equal(y, linear(x, p))


# every tile of the GEMM, with rows and columns that end inside one
TILES = [(513, 192, 500), (1100, 128, 2100), (1900, 64, 2000), (2100, 128, 2001),
         (2900, 64, 2400), (3, 64, 9000), (17, 128, 9000), (33, 192, 6000), (64, 100, 4500), (3000, 192, 3900), (4200, 128, 4001),
         (5400, 64, 5290)]  # fmt: skip


@pytest.mark.parametrize("weights,rows", [("bf16", "bf16"), ("w8c", "bf16"), ("w8c", "q8")])
@pytest.mark.parametrize("T,K,N", TILES)
def test_every_tile(dev, T, K, N, weights, rows):
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    x, w, xd, wd = make(dev, T, K, N, weights, rows)
    p = prepack_linear(w)
    check(linear(x, p), xd, wd, K)
    L, R = 7, 40
    lora = make_adapters(dev, T, K, N, L, R)
    y = linear(x, p, lora=prepack_lora(*lora[:3]), batch=lora_batch(lora[3], L))
    check(y, xd, wd, K, lora, R)


LORA = [
    # T, K, N, L, R
    (1, 64, 16, 1, 1), (1, 2048, 512, 4, 16), (5, 100, 31, 3, 8), (16, 256, 130, 16, 64), (33, 192, 64, 5, 33),
    (64, 1024, 96, 32, 16), (64, 128, 40, 2, 256), (65, 64, 16, 1, 1), (66, 256, 128, 70, 16), (130, 1000, 257, 3, 24),
    (257, 320, 130, 9, 64), (300, 512, 1000, 300, 8), (333, 128, 40, 2, 256), (1000, 2048, 384, 5, 32),
]  # fmt: skip


@pytest.mark.parametrize("weights,rows", [("bf16", "bf16"), ("w8c", "bf16"), ("w8c", "q8")])
@pytest.mark.parametrize("T,K,N,L,R", LORA)
def test_lora(dev, T, K, N, L, R, weights, rows):
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    x, w, xd, wd = make(dev, T, K, N, weights, rows)
    lora = make_adapters(dev, T, K, N, L, R)
    p, l, batch = prepack_linear(w), prepack_lora(*lora[:3]), lora_batch(lora[3], L)
    y = linear(x, p, lora=l, batch=batch)
    check(y, xd, wd, K, lora, R)
    assert torch.equal(y, linear(x, p, lora=l, batch=batch))
    if T > 64:  # (smaller batches sum in another order beside adapters)
        none = torch.nonzero(lora[3] < 0).squeeze(1)
        assert torch.equal(y[none], linear(x, p)[none])


@pytest.mark.parametrize("T", [40, 400])
def test_adapters_of_requests_side_by_side(dev, T):
    """Requests of several tokens, one of them without an adapter; all tokens of one adapter;
    none of any."""
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    K, N, L, R = 512, 320, 6, 16
    x, w, xd, wd = make(dev, T, K, N)
    a, b, f, _ = make_adapters(dev, T, K, N, L, R)
    p, l = prepack_linear(w), prepack_lora(a, b, f)
    cut = torch.arange(T, device=dev)
    for ad in (
        torch.where(cut < T // 3, 5, torch.where(cut < T // 2, -1, 2)), torch.full((T,), 3, device=dev),
        torch.full((T,), -1, device=dev), cut % L, torch.full((T,), L, device=dev), torch.full((T,), 2**40, device=dev),
    ):  # fmt: skip
        y = linear(x, p, lora=l, batch=lora_batch(ad, L))
        check(y, xd, wd, K, (a, b, f, ad), R)


@pytest.mark.parametrize("T,L", [(1, 1), (64, 7), (511, 64), (512, 3), (513, 1024), (2000, 7), (5000, 300)])
def test_lora_batch_is_a_stable_sort(dev, T, L):
    from kappa_amd.qwen3 import lora_batch

    g = _gen(dev, T, L)
    ad = torch.randint(-3, L + 3, (T,), generator=g, device=dev).to(torch.int32)
    bt = lora_batch(ad, L)
    bucket = torch.where((ad >= 0) & (ad < L), ad, torch.full_like(ad, L)).cpu()
    order = torch.argsort(bucket, stable=True)
    got = bt.buffer.cpu()
    clean = torch.where(bucket == L, torch.full_like(bucket, -1), bucket)
    assert torch.equal(got[:T], clean)
    assert torch.equal(got[T : 2 * T], order.to(torch.int32))
    assert torch.equal(got[2 * T : 3 * T], clean[order])
    starts = torch.cumsum(torch.bincount(bucket, minlength=L + 1), 0) - torch.bincount(bucket, minlength=L + 1)
    assert torch.equal(got[3 * T : 3 * T + L + 1], starts.to(torch.int32))


@pytest.mark.parametrize("T", [8, 200])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_what_is_not_finite_stays_in_its_rows(dev, T, bad):
    """An adapter whose values overflowed, and a row that did, leave the other rows their bits."""
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    K, N, L, R = 256, 160, 3, 16
    x, w, xd, wd = make(dev, T, K, N, "bf16")
    a, b, f, _ = make_adapters(dev, T, K, N, L, R)
    ad = (torch.arange(T, device=dev) % (L + 1) - 1).to(torch.int32)
    p = prepack_linear(w)
    want = linear(x, p, lora=prepack_lora(a, b, f), batch=lora_batch(ad, L))
    b2 = b.clone()
    b2[1, 3, 7] = bad
    y = linear(x, p, lora=prepack_lora(a, b2, f), batch=lora_batch(ad, L))
    other = ad != 1
    assert torch.equal(y[other], want[other])
    assert not torch.isfinite(y[~other][:, 7]).any()
    x2 = x.clone()
    x2[3, 5] = bad
    y = linear(x2, p, lora=prepack_lora(a, b, f), batch=lora_batch(ad, L))
    other = torch.arange(T, device=dev) != 3
    assert torch.equal(y[other], want[other]) and not torch.isfinite(y[3]).any()


@pytest.mark.parametrize("T,K,N", [(8, 256, 96), (100, 256, 96), (300, 192, 1000), (700, 128, 2600), (2900, 64, 2400)])
@pytest.mark.parametrize("R", [16, 70])
def test_a_row_keeps_its_bits_whatever_its_neighbours_take(dev, T, K, N, R):
    """The adapters of every third token stay, those of the others change (all of one, one
    each, none): the sorted order, the tiles' ranges and the neighbours do, the row does not."""
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    L = 40
    x, w, _, _ = make(dev, T, K, N)
    a, b, f, ad = make_adapters(dev, T, K, N, L, R)
    p, l = prepack_linear(w), prepack_lora(a, b, f)
    t = torch.arange(T, device=dev)
    stay = t % 3 == 0
    want = linear(x, p, lora=l, batch=lora_batch(ad, L))[stay]
    for other in (torch.full_like(ad, 5), (t % L).to(ad.dtype), torch.full_like(ad, -1)):
        y = linear(x, p, lora=l, batch=lora_batch(torch.where(stay, ad, other), L))
        assert torch.equal(y[stay], want)


@pytest.mark.parametrize("T", [6, 90])
@pytest.mark.parametrize("rows", ["bf16", "q8"])
def test_rows_of_other_layouts(dev, T, rows):
    """Strided rows, rows off 16-byte boundaries, columns apart, more axes."""
    from kappa_amd.qwen3 import Q8Rows, linear, prepack_linear

    K, N = 256, 96
    x, w, xd, wd = make(dev, T, K, N, "w8c", rows)
    p = prepack_linear(w)
    v = x.values if rows == "q8" else x
    wrap = (lambda t: Q8Rows(t, x.scale)) if rows == "q8" else (lambda t: t)
    y = linear(x, p)
    wide = torch.zeros(T, K + 64, dtype=v.dtype, device=dev)
    wide[:, 16 : 16 + K] = v
    assert torch.equal(linear(wrap(wide[:, 16 : 16 + K]), p), y)
    odd = torch.zeros(T, K + 3, dtype=v.dtype, device=dev)
    odd[:, 1 : 1 + K] = v
    assert torch.equal(linear(wrap(odd[:, 1 : 1 + K]), p), y)
    assert torch.equal(linear(wrap(v.t().contiguous().t()), p), y)
    three = linear(wrap(v.view(2, T // 2, K)), p)
    assert three.shape == (2, T // 2, N) and torch.equal(three.view(T, N), y)
    same = v[:1].expand(T, K)
    if rows == "bf16":
        assert torch.equal(linear(same, p), y[:1].expand(T, N))
    one = linear(Q8Rows(v[0], x.scale[0]) if rows == "q8" else v[0], p)
    assert one.shape == (N,)
    check(one.view(1, N), xd[:1], wd, K)


def test_slots_are_stored_one_by_one(dev):
    """LoraAdapters.empty adds nothing; store fills slots, with smaller ranks too, and leaves the others."""
    from kappa_amd.qwen3 import LoraAdapters, linear, lora_batch, prepack_linear

    T, K, N, L = 30, 192, 72, 4
    x, w, xd, wd = make(dev, T, K, N)
    p = prepack_linear(w)
    ad = (torch.arange(T, device=dev) % L).to(torch.int32)
    batch = lora_batch(ad, L)
    slots = LoraAdapters.empty(L, 40, K, N, device=dev)
    check(linear(x, p, lora=slots, batch=batch), xd, wd, K)
    a, b, f, _ = make_adapters(dev, T, K, N, L, 40)
    slots.store(0, a, b, f)
    check(linear(x, p, lora=slots, batch=batch), xd, wd, K, (a, b, f, ad), 40)
    a2, b2 = a[:1, :, :7].contiguous(), b[:1, :7].contiguous()
    slots.store(2, a2[0], b2[0], 0.5)
    a[2], b[2], f[2] = 0, 0, 0.5
    a[2, :, :7], b[2, :7] = a2[0], b2[0]
    check(linear(x, p, lora=slots, batch=batch), xd, wd, K, (a, b, f, ad), 40)


def test_packed_weights_are_copied_whole(dev):
    """Copies and replaced fields call the kernels with their own buffers."""
    import copy
    import dataclasses
    import pickle

    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    T, K, N, L, R = 9, 128, 64, 2, 8
    x, w, xd, wd = make(dev, T, K, N)
    _, w2, _, wd2 = make(dev, T, K, N, seed=1)
    lora = make_adapters(dev, T, K, N, L, R)
    p, p2, l, batch = prepack_linear(w), prepack_linear(w2), prepack_lora(*lora[:3]), lora_batch(lora[3], L)
    want = linear(x, p, lora=l, batch=batch)
    pc, lc, bc = copy.deepcopy(p), copy.deepcopy(l), pickle.loads(pickle.dumps(batch))
    other = dataclasses.replace(p, values=p2.values, scale=p2.scale)
    p.values.zero_()
    l.a.zero_()
    batch.buffer.zero_()
    assert torch.equal(linear(x, pc, lora=lc, batch=bc), want)
    check(linear(x, other), xd, wd2, K)


@pytest.mark.parametrize("T", [0, 3, 70])
def test_nothing_behind_the_last_row_is_written(dev, T):
    from kappa_amd import _lib
    from kappa_amd.qwen3 import prepack_linear
    from kappa_amd.qwen3.projection import _stream

    K, N = 128, 45
    x, w, xd, wd = make(dev, T, K, N)
    p = prepack_linear(w)
    out = torch.full((T * N + 64,), 7.0, dtype=torch.bfloat16, device=dev)
    n = ctypes.c_size_t()
    L = _lib.lib()
    _lib.check(L.kmoe_linear_workspace_bytes(p.struct, T, _lib.DTYPE_BF16, None, ctypes.byref(n)))
    ws = torch.empty(n.value + 16, dtype=torch.uint8, device=dev)
    _lib.check(L.kmoe_linear(p.struct, T, x.data_ptr(), _lib.DTYPE_BF16, K, None, None, None, out.data_ptr(),
                             ws.data_ptr(), n.value, _stream(dev)))  # fmt: skip
    check(out[: T * N].view(T, N), xd, wd, K)
    assert (out[T * N :] == 7.0).all()


@pytest.mark.parametrize("T", [24, 150])
def test_a_step_in_a_graph(dev, T):
    """The sort, two projections and the norms of a step, captured; the tokens' adapters, the
    rows and a slot change between replays."""
    from kappa_amd.qwen3 import LoraAdapters, add_rms_norm, add_rms_norm_q8, linear, lora_batch, prepack_linear

    K, L, R = 512, 5, 16
    _, w1, _, _ = make(dev, T, K, 768)
    _, w2, _, _ = make(dev, T, 768, K)
    p1, p2 = prepack_linear(w1), prepack_linear(w2)
    a1, b1, f1, ad = make_adapters(dev, T, K, 768, L, R)
    a2, b2, f2, _ = make_adapters(dev, T, 768, K, L, R)
    l1, l2 = LoraAdapters.empty(L, R, K, 768, device=dev), LoraAdapters.empty(L, R, 768, K, device=dev)
    l1.store(0, a1, b1, f1)
    l2.store(0, a2, b2, f2)
    g = _gen(dev, T)
    x, res = _randn(g, dev, T, K), _randn(g, dev, T, K)
    scale = torch.ones(K, dtype=torch.bfloat16, device=dev)

    def step():
        batch = lora_batch(ad, L)
        n, h = add_rms_norm(x, res, scale)
        y = linear(linear(n, p1, lora=l1, batch=batch), p2, lora=l2, batch=batch)
        q, h = add_rms_norm_q8(y, h, scale)
        return linear(q, p1, lora=l1, batch=batch), h

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gh = step()
    for k in range(4):
        x.copy_(_randn(g, dev, T, K))
        ad.copy_(torch.randint(-1, L, (T,), generator=g, device=dev))
        if k == 2:
            l1.store(1, _randn(g, dev, K, 4, std=0.1), _randn(g, dev, 4, 768), 2.0)
        graph.replay()
        y, h = step()
        torch.cuda.synchronize()
        assert torch.equal(gy, y) and torch.equal(gh, h), k


def test_two_streams_at_once(dev):
    from kappa_amd.qwen3 import linear, lora_batch, prepack_linear, prepack_lora

    T, K, N, L, R = 100, 1024, 512, 4, 16
    x, w, _, _ = make(dev, T, K, N)
    x2 = make(dev, T, K, N, seed=1)[0]
    lora = make_adapters(dev, T, K, N, L, R)
    p, l, batch = prepack_linear(w), prepack_lora(*lora[:3]), lora_batch(lora[3], L)
    want = [linear(t, p, lora=l, batch=batch) for t in (x, x2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(linear((x, x2)[k], p, lora=l, batch=batch))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in got[k])


@pytest.mark.parametrize("T", [4, 96])
@pytest.mark.parametrize("rows", ["bf16", "q8"])
def test_a_layer_of_them(dev, T, rows):
    """From the MoE half of one layer to the heads of the next, against 64 bits: the block's
    output, the residual and norm, the projection with adapters."""
    from kappa_amd.qwen3 import (
        Q8Weight, add_rms_norm, add_rms_norm_q8, linear, lora_batch, moe_block_ffn, moe_layer_config, prepack_linear,
        prepack_lora, quantize_weight_per_channel,
    )  # fmt: skip

    D, E, I, N, L, R = 256, 16, 128, 384, 3, 8
    g = _gen(dev, T, rows)
    cfg = moe_layer_config(hidden=D, experts=E, top_k=4, intermediate=I, moe_impl="ragged_jax",
                           moe_ragged_decode_token_threshold=0)  # fmt: skip
    h0 = _randn(g, dev, 1, T, D)
    router = _randn(g, dev, D, E, std=0.05)
    ws = [quantize_weight_per_channel(_randn(g, dev, *s, std=0.05)) for s in ((E, D, I), (E, D, I), (E, I, D))]
    scale = (1.0 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16)
    w = quantize_weight_per_channel(_randn(g, dev, D, N, std=D**-0.5))
    assert isinstance(w, Q8Weight)
    p = prepack_linear(w)
    a, b, f, ad = make_adapters(dev, T, D, N, L, R)
    l, batch = prepack_lora(a, b, f), lora_batch(ad, L)
    x = moe_block_ffn(h0, scale, router, *ws, cfg=cfg)
    attn = _randn(g, dev, 1, T, D)
    n, h = (add_rms_norm_q8 if rows == "q8" else add_rms_norm)(attn, x, scale)
    y = linear(n, p, lora=l, batch=batch)
    assert y.shape == (1, T, N) and torch.equal(h, attn + x)
    # the projection's own error, from the rows as they are
    nd = n.values.double() * n.scale.double() if rows == "q8" else n.double()
    check(y[0], nd[0], w.values.double() * w.scale.double(), D, (a, b, f, ad), R)
    # and the rows' from the formula: half a step of 8 bits of the largest, or of bf16
    hd = h[0].double()
    v = hd / torch.sqrt((hd * hd).mean(dim=1, keepdim=True) + 1e-6) * scale.double()
    tol = v.abs().amax(dim=1, keepdim=True) / 254 * (1 + 1e-3) if rows == "q8" else v.abs() * 2.0**-8 * (1 + 1e-3)
    assert ((nd[0] - v).abs() <= tol).all()


def test_refusals(dev):
    from kappa_amd.qwen3 import (
        LoraAdapters, Q8Rows, Q8Weight, linear, lora_batch, prepack_linear, prepack_lora,
    )  # fmt: skip

    T, K, N, L, R = 4, 128, 64, 2, 8
    x, w, _, _ = make(dev, T, K, N)
    xb, wb, _, _ = make(dev, T, K, N, "bf16")
    p, pb = prepack_linear(w), prepack_linear(wb)
    a, b, f, ad = make_adapters(dev, T, K, N, L, R)
    l, batch = prepack_lora(a, b, f), lora_batch(ad, L)
    q = Q8Rows(torch.zeros(T, K, dtype=torch.int8, device=dev), torch.ones(T, 1, device=dev))

    def refused(match, call, *args, **kw):
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)

    refused("must be a PackedLinear", linear, x, w)
    refused("bfloat16 or Q8Rows", linear, x.float(), p)
    refused("rows of 128", linear, x[:, :64], p)
    refused("int8 weights", linear, q, pb)
    refused("one per row", linear, Q8Rows(q.values, q.scale[:3]), p)
    refused("int8 with float32", linear, Q8Rows(q.values, q.scale.half()), p)
    refused("x is on", linear, x.cpu(), p)
    refused("come together", linear, x, p, lora=l)
    refused("must be LoraAdapters", linear, x, p, lora=(a, b), batch=batch)
    refused("tokens", linear, x[:3], p, lora=l, batch=batch)
    refused("adapters", linear, x, p, lora=l, batch=lora_batch(ad, L + 1))
    other = prepack_lora(a, b[:, :, :32].contiguous(), f)
    refused("the weights", linear, x, p, lora=other, batch=batch)
    refused("bfloat16 or a Q8Weight", prepack_linear, wb.float())
    refused(r"\[in, out\]", prepack_linear, wb[0])
    refused("neither a scalar nor per output channel", prepack_linear, Q8Weight(w.values, torch.ones(N + 1, device=dev)))
    refused("HIP device", prepack_linear, wb.cpu())
    refused("must be int32", lora_batch, ad.float(), L)
    refused("exceeds 1024", lora_batch, ad, 1025)
    refused("num_adapters must be", lora_batch, ad, 0)
    refused("exceeds 256", LoraAdapters.empty, 2, 257, K, N)
    refused("slots", l.store, 1, a, b, f)
    refused("slots", l.store, -1, a[:1], b[:1], 1.0)
    refused("rank 8 is not", LoraAdapters.empty(2, 4, K, N, device=dev).store, 0, a, b, f)
    refused("must be bfloat16", l.store, 0, a.float(), b, f)
    refused("entries for", l.store, 0, a, b, f[:1])
    refused("are not", l.store, 0, a[:, :64], b, f)
