"""add_rms_norm and add_rms_norm_q8 (GPU): the residual's addition with the norm after it.

add_rms_norm promises the bits of the two steps it replaces, x + residual rounded to the
activation type and rms_norm of that. The 8-bit form is compared with its formula in 64
bits: v = (h r) g in f32 is off by at most three roundings and the relative error of r,
which the f32 sum of D squares gives ((D + 4) 2^-24 at most, halved by the root)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
TINY = torch.finfo(torch.float32).tiny


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    return torch.device("cuda:0")


def _case(dev, T, D, act, sdt, seed=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + T * 31 + D)
    x = torch.randn(T, D, generator=g, device=dev).to(DTYPES[act])
    res = (3.0 * torch.randn(T, D, generator=g, device=dev)).to(DTYPES[act])
    scale = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(DTYPES[sdt])
    return x, res, scale


def _misaligned(t):
    """The same values, one element off the 16-byte boundary."""
    buf = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    v = buf[1 : 1 + t.numel()].view(t.shape)
    v.copy_(t)
    return v


SHAPES = [(1003, 64), (1500, 1000), (2049, 512), (1, 1), (3, 63), (2, 64), (5, 100), (1, 1024), (4, 2048), (257, 2048), (33, 2560), (1, 4096), (70, 4096), (9, 4095)]


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("sdt", ["bf16", "f32"])
@pytest.mark.parametrize("T,D", SHAPES)
def test_add_rms_norm_has_the_bits_of_the_two_steps(dev, T, D, act, sdt):
    from kappa_amd.qwen3 import add_rms_norm, rms_norm

    x, res, scale = _case(dev, T, D, act, sdt)
    normed, h = add_rms_norm(x, res, scale, epsilon=EPS)
    want = (x.float() + res.float()).to(x.dtype)
    assert torch.equal(h, want)
    assert torch.equal(normed, rms_norm(want, scale, epsilon=EPS))


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("D", [128, 2048, 100])
def test_add_rms_norm_of_views(dev, D, act):
    """Buffers off 16-byte boundaries, transposed ones, and more axes."""
    from kappa_amd.qwen3 import add_rms_norm, add_rms_norm_q8

    x, res, scale = _case(dev, 6, D, act, "bf16", 1)
    normed, h = add_rms_norm(x, res, scale)
    q, _ = add_rms_norm_q8(x, res, scale)
    for xs, rs, ss in (
        (_misaligned(x), res, scale), (x, _misaligned(res), scale), (x, res, _misaligned(scale)),
        (x.t().contiguous().t(), res, scale),
    ):  # fmt: skip
        n2, h2 = add_rms_norm(xs, rs, ss)
        assert torch.equal(n2, normed) and torch.equal(h2, h)
        q2, h3 = add_rms_norm_q8(xs, rs, ss)
        assert torch.equal(q2.values, q.values) and torch.equal(q2.scale, q.scale) and torch.equal(h3, h)
    n3, h3 = add_rms_norm(x.view(2, 3, D), res.view(2, 3, D), scale)
    assert n3.shape == (2, 3, D) and torch.equal(n3.view(6, D), normed) and torch.equal(h3.view(6, D), h)
    q3, _ = add_rms_norm_q8(x.view(2, 3, D), res.view(2, 3, D), scale)
    assert q3.values.shape == (2, 3, D) and q3.scale.shape == (2, 3, 1)


def _check_q8(h, scale, q, D):
    """h: the summed rows; q: Q8Rows. Rows must be finite."""
    hd = h.double()
    v = hd / torch.sqrt((hd * hd).sum(dim=1, keepdim=True) / D + EPS) * scale.double()
    rel = 0.5 * (D + 4) * 2.0**-24 + 5 * 2.0**-24
    want = torch.clamp_min(v.abs().amax(dim=1, keepdim=True) / 127.0, TINY)
    assert ((q.scale.double() - want).abs() <= want * (rel + 2.0**-23)).all()
    # the nearest integer of v / scale, up to the error of v, of the scale, of 1 / scale and of the product
    off = (q.values.double() - v / want).abs()
    assert (off <= 0.5 + 127.0 * (2 * rel + 4 * 2.0**-24)).all(), float(off.max())
    assert int(q.values.abs().max()) <= 127


@pytest.mark.parametrize("act", ["bf16", "f32"])
@pytest.mark.parametrize("T,D", SHAPES)
def test_q8_against_the_formula(dev, T, D, act):
    from kappa_amd.qwen3 import add_rms_norm_q8

    x, res, scale = _case(dev, T, D, act, "bf16", 2)
    q, h = add_rms_norm_q8(x, res, scale, epsilon=EPS)
    assert torch.equal(h, (x.float() + res.float()).to(x.dtype))
    _check_q8(h, scale, q, D)
    q2, h2 = add_rms_norm_q8(h, None, scale, epsilon=EPS)
    assert h2 is h and torch.equal(q2.values, q.values) and torch.equal(q2.scale, q.scale)


@pytest.mark.parametrize("T,D,act", [(2048, 4096, "bf16"), (1024, 4096, "f32"), (17000, 500, "bf16"), (9, 4095, "bf16")])
def test_q8_is_the_rounded_quotient(dev, T, D, act):
    """Bit for bit rint(v / s): v in f32 is what rms_norm gives for the same rows in float32,
    the division rounds once (done here on the CPU)."""
    from kappa_amd.qwen3 import add_rms_norm_q8, rms_norm

    x, res, scale = _case(dev, T, D, act, "bf16", 8)
    if act == "f32":  # every fourth row so small that its scale is near, or at, the smallest float
        x[::4] *= 2.0**-113
        res[::4] *= 2.0**-113
        x[::8] *= 2.0**-8
        res[::8] *= 2.0**-8
    q, h = add_rms_norm_q8(x, res, scale, epsilon=EPS)
    v = rms_norm(h.float(), scale.float(), epsilon=EPS).cpu()
    s = torch.clamp_min(v.abs().amax(dim=1, keepdim=True) / 127.0, TINY)
    assert torch.equal(q.scale.cpu(), s)
    want = torch.clamp(torch.round(v / s), -127.0, 127.0)
    got = q.values.cpu().float()
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("D", [128, 100, 4096])
def test_q8_rows_at_the_edges(dev, D):
    """Zero rows, tiny rows, and rows with an infinity or a NaN, beside an ordinary one."""
    from kappa_amd.qwen3 import add_rms_norm_q8

    x, res, scale = _case(dev, 6, D, "f32", "f32", 3)
    res[1:] = 0.0
    x[1] = 0.0
    x[2] *= 1e-30
    x[3, D // 2] = float("inf")
    x[4, D - 1] = float("nan")
    x[5, 0] = -float("inf")
    q, h = add_rms_norm_q8(x, res, scale, epsilon=EPS)
    _check_q8(h[:1], scale, q.__class__(q.values[:1], q.scale[:1]), D)
    assert float(q.scale[1]) == TINY and not q.values[1].any()
    # epsilon keeps the norm of row 2 near 1e-27: still full 8 bits
    _check_q8(h[2:3], scale, q.__class__(q.values[2:3], q.scale[2:3]), D)
    assert torch.isnan(q.scale[3:]).all() and not q.values[3:].any()


def test_in_place(dev):
    """h_out may be x or residual (C ABI)."""
    from kappa_amd import _lib
    from kappa_amd.qwen3 import add_rms_norm, add_rms_norm_q8
    from kappa_amd.qwen3.ffn_moe import _desc, _stream

    for D in (2048, 100):
        x, res, scale = _case(dev, 37, D, "bf16", "bf16", 4)
        normed, h = add_rms_norm(x, res, scale)
        q, _ = add_rms_norm_q8(x, res, scale)
        for which in (0, 1):
            a, b = x.clone(), res.clone()
            out = torch.empty_like(x)
            at = (a, b)[which]
            d = _desc(37, D, 1, 1, 1, x.dtype)
            _lib.check(_lib.lib().kmoe_add_rms_norm(d, a.data_ptr(), b.data_ptr(), scale.data_ptr(), _lib.DTYPE_BF16,
                                                    EPS, at.data_ptr(), out.data_ptr(), _stream(dev)))  # fmt: skip
            assert torch.equal(at, h) and torch.equal(out, normed)
            a, b = x.clone(), res.clone()
            at = (a, b)[which]
            qv, qs = torch.empty_like(q.values), torch.empty_like(q.scale)
            _lib.check(_lib.lib().kmoe_add_rms_norm_q8(d, a.data_ptr(), b.data_ptr(), scale.data_ptr(),
                                                       _lib.DTYPE_BF16, EPS, at.data_ptr(), qv.data_ptr(),
                                                       qs.data_ptr(), _stream(dev)))  # fmt: skip
            assert torch.equal(at, h) and torch.equal(qv, q.values) and torch.equal(qs, q.scale)


@pytest.mark.parametrize("T,D", [((1 << 24) + 5, 1032), ((1 << 26) + 5, 8)])
def test_more_rows_than_one_launch_takes(dev, T, D):
    """A launch holds less than 2^32 threads: 2^24 rows of 256, 2^26 of 64. Rows repeat after 1009."""
    from kappa_amd.qwen3 import add_rms_norm, add_rms_norm_q8, rms_norm

    x, res, scale = _case(dev, 1009, D, "bf16", "bf16", 9)
    many = x.repeat(-(-T // 1009), 1)[:T]
    q, s = add_rms_norm_q8(many, None, scale)[0]
    want = add_rms_norm_q8(x, None, scale)[0]
    for t in (0, 12345, T - 2018 - T % 1009, T - 1009 - T % 1009):
        a = -t % 1009 + t  # where the pattern starts
        n = min(1009, T - a)
        assert torch.equal(q[a : a + n], want.values[:n]) and torch.equal(s[a : a + n], want.scale[:n])
    n = T % 1009
    assert torch.equal(q[T - n :], want.values[:n]) and torch.equal(s[T - n :], want.scale[:n])
    if D == 8:
        normed, h = add_rms_norm(many, res.repeat(-(-T // 1009), 1)[:T], scale)
        want, hw = add_rms_norm(x, res, scale)
        assert torch.equal(normed[T - n :], want[:n]) and torch.equal(h[T - n :], hw[:n])
        assert torch.equal(normed[:1009], want) and torch.equal(h[:1009], hw)
        normed, want = rms_norm(many, scale), rms_norm(x, scale)
        assert torch.equal(normed[T - n :], want[:n]) and torch.equal(normed[:1009], want)


def test_no_rows(dev):
    from kappa_amd.qwen3 import add_rms_norm, add_rms_norm_q8

    x = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    scale = torch.ones(64, dtype=torch.bfloat16, device=dev)
    normed, h = add_rms_norm(x, x, scale)
    assert normed.shape == h.shape == (0, 64)
    q, _ = add_rms_norm_q8(x, x, scale)
    assert q.values.shape == (0, 64) and q.scale.shape == (0, 1)


def test_on_another_stream_and_in_a_graph(dev):
    from kappa_amd.qwen3 import add_rms_norm, add_rms_norm_q8

    x, res, scale = _case(dev, 64, 2048, "bf16", "bf16", 5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        n1, h1 = add_rms_norm(x, res, scale)
        q1, _ = add_rms_norm_q8(x, res, scale)
    torch.cuda.current_stream().wait_stream(s)
    n, h = add_rms_norm(x, res, scale)
    q, _ = add_rms_norm_q8(x, res, scale)
    assert torch.equal(n, n1) and torch.equal(h, h1) and torch.equal(q.values, q1.values)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gn, gh = add_rms_norm(x, res, scale)
        gq, _ = add_rms_norm_q8(gh, None, scale)
    for k in range(3):
        x.copy_(torch.randn_like(x))
        g.replay()
        n, h = add_rms_norm(x, res, scale)
        q, _ = add_rms_norm_q8(x, res, scale)
        torch.cuda.synchronize()
        assert torch.equal(gn, n) and torch.equal(gh, h) and torch.equal(gq.values, q.values), k
        assert torch.equal(gq.scale, q.scale)


def test_refusals(dev):
    from kappa_amd.qwen3 import add_rms_norm, add_rms_norm_q8

    x, res, scale = _case(dev, 4, 64, "bf16", "bf16", 6)
    with pytest.raises(ValueError, match="needs a residual"):
        add_rms_norm(x, None, scale)
    with pytest.raises(ValueError, match="residual must be as x"):
        add_rms_norm(x, res[:3], scale)
    with pytest.raises(ValueError, match="residual must be as x"):
        add_rms_norm_q8(x, res.float(), scale)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        add_rms_norm(x.half(), res.half(), scale)
    with pytest.raises(ValueError, match="norm scale has"):
        add_rms_norm(x, res, scale[:63])
    with pytest.raises(ValueError, match="epsilon"):
        add_rms_norm(x, res, scale, epsilon=-1.0)
    with pytest.raises(ValueError, match="HIP device"):
        add_rms_norm_q8(x.cpu(), None, scale)
    big = torch.zeros(1, 4097, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="hidden 4097"):
        add_rms_norm(big, big, torch.ones(4097, device=dev))
