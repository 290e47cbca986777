"""e2mi_rope against the rotation in 64 bits, its gradient, its strides and orders of use.

Tolerance: with a sine and a cosine off by at most 2 steps of 2^-24 and the rounded angle by 2^-28 turns
(0.4 steps), the magnitude's and each product's rounding one step each, a value is off by at most 8 * 2^-24 *
m * (|x1| + |x2|) before its rounding to the output type, half a step of the value (for f16 never under half
of its smallest subnormal, 2^-25)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def _want(x, pos, freqs, n, layout, mag, inverse):
    """y and its tolerance per value, from x [M, n * D] (64-bit values of the inputs)."""
    import torch
    M = x.shape[0]
    v = x.double().cpu().view(M, n, -1)
    half = freqs.numel()
    a = pos.cpu().double()[:, None] * freqs.cpu()[None]
    # a product of a position below 2^31 and a frequency: 64 bits leave 2^-22 rad at 10^9 rad; positions
    # here stay under 2^22, where that is 2^-31
    c, s = (mag * a.cos())[:, None], (mag * (-a if inverse else a).sin())[:, None]
    i = torch.arange(half)
    lo, hi = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    y, t = v.clone(), torch.zeros_like(v)
    y[..., lo] = v[..., lo] * c - v[..., hi] * s
    y[..., hi] = v[..., hi] * c + v[..., lo] * s
    size = 8 * 2.0 ** -24 * abs(mag) * (v[..., lo].abs() + v[..., hi].abs())
    t[..., lo] = size
    t[..., hi] = size
    return y.view(M, -1), t.view(M, -1)


def _check(got, x, pos, freqs, n, layout, mag=1.0, inverse=False):
    y, t = _want(x, pos, freqs, n, layout, mag, inverse)
    kind = str(got.dtype).replace("torch.", "")
    tol = t + EPS[kind] * (y.abs() + t) + (2.0 ** -25 if kind == "float16" else 0.0)
    off = (got.double().cpu() - y).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("M,H,KV,D,rot", [
    (1, 3, 1, 256, 256),     # one token
    (37, 4, 2, 256, 128),    # part of the head, whole 16-byte chunks
    (5, 2, 1, 64, 18),       # part of the head, no whole chunks
    (130, 16, 4, 128, 128),
    (3, 1, 1, 512, 512),
    (9, 2, 2, 6, 2),         # one pair, a head of no 16-byte size
    (2051, 3, 1, 256, 256),  # enough rows for a thread to walk all heads
])
def test_rotation(gpu, dtype, layout, M, H, KV, D, rot):
    import e2mi
    import torch
    t = getattr(torch, dtype)
    g = torch.Generator(device=gpu).manual_seed(M * 7 + rot)
    q = torch.randn((M, H * D), generator=g, device=gpu).to(t)
    k = (3.0 * torch.randn((M, KV * D), generator=g, device=gpu)).to(t)
    pos = torch.randint(-1000, 1 << 22, (M,), generator=g, device=gpu, dtype=torch.int32)
    freqs = e2mi.rope_freqs(rot, 10000.0, "parts", 4.0, trained_len=4096).to(gpu)
    for mag, inverse in ((1.0, False), (1.1386, True)):
        qo, ko = e2mi.rope(q, k, pos, freqs, H, KV, layout=layout, magnitude=mag, inverse=inverse)
        m32 = float(np.float32(mag))
        _check(qo, q, pos, freqs, H, layout, m32, inverse)
        _check(ko, k, pos, freqs, KV, layout, m32, inverse)


def test_far_positions(gpu):
    """Positions to the ends of int32: angles against integers of turns, f_i = 2 pi / 2^i exactly as many
    turns as the position has 2^i (the f64 frequency's rounding moves 2^31 of them by 2^-22 turns)."""
    import e2mi
    import torch
    pos = torch.tensor([-2 ** 31, -2 ** 31 + 1, 2 ** 31 - 1, 2 ** 30 + 3, 123456789, 0], dtype=torch.int32, device=gpu)
    i = torch.arange(4)
    freqs = (2 * np.pi / 2.0 ** (i.double() + 2)).to(gpu)  # turns = pos / 4, / 8, / 16, / 32
    x = torch.zeros((6, 8), dtype=torch.float32, device=gpu)
    x[:, :4] = 1.0
    y, _ = e2mi.rope(x, None, pos, freqs, 1, 0)
    for r in range(6):
        for j in range(4):
            a = 2 * np.pi * (int(pos[r]) % 2 ** (j + 2)) / 2 ** (j + 2)
            assert abs(float(y[r, j]) - np.cos(a)) <= 2 * np.pi * 2.0 ** -22 + 2.0 ** -21
            assert abs(float(y[r, 4 + j]) - np.sin(a)) <= 2 * np.pi * 2.0 ** -22 + 2.0 ** -21


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_strided_and_sides(gpu, layout):
    """q and k as columns of one fused row buffer, turned in place: the values beside them stay; q alone and k
    alone give the same; the inverse takes them back."""
    import e2mi
    import torch
    M, H, KV, D, rot = 29, 3, 1, 128, 64
    g = torch.Generator(device=gpu).manual_seed(3)
    row = torch.randn((M, (H + 2 * KV) * D + 8), generator=g, device=gpu)
    was = row.clone()
    q, k = row[:, :H * D], row[:, H * D:(H + KV) * D]
    pos = torch.arange(M, dtype=torch.int32, device=gpu) * 977
    freqs = e2mi.rope_freqs(rot).to(gpu)
    want_q, _ = e2mi.rope(q, None, pos, freqs, H, 0, layout=layout)
    _, want_k = e2mi.rope(None, k, pos, freqs, 0, KV, layout=layout)
    e2mi.rope(q, k, pos, freqs, H, KV, layout=layout, q_out=q, k_out=k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(row[:, (H + KV) * D:], was[:, (H + KV) * D:])
    _check(want_q, was[:, :H * D], pos, freqs, H, layout)
    e2mi.rope(q, k, pos, freqs, H, KV, layout=layout, q_out=q, k_out=k, inverse=True)
    # there and back: each way off by 8 * 2^-24 (|x1| + |x2|) + half a step
    assert float((row - was).abs().max()) <= 2 * 10 * 2.0 ** -24 * 2 * float(was.abs().max())
    # rows that start off 16 bytes take the element-wise kernel, with the same angles and values
    off = torch.empty(M, H * D + 3, device=gpu)[:, 3:]
    off.copy_(was[:, :H * D])
    got, _ = e2mi.rope(off, None, pos, freqs, H, 0, layout=layout)
    assert torch.equal(got, want_q)


def test_gradient(gpu):
    """inverse is the transpose: <rope(x), g> = <x, rope^-1(g)>, and against differences of the forward."""
    import e2mi
    import torch
    M, H, D = 4, 2, 64
    g0 = torch.Generator(device=gpu).manual_seed(11)
    x, g = (torch.randn((M, H * D), generator=g0, device=gpu) for _ in range(2))
    pos = torch.tensor([0, 5, 4097, 70001], dtype=torch.int32, device=gpu)
    freqs = e2mi.rope_freqs(48, 10000.0, "base", 8.0).to(gpu)
    f = lambda v, inv=False: e2mi.rope(v, None, pos, freqs, H, 0, layout="interleaved", magnitude=1.25, inverse=inv)[0]  # noqa: E731
    y, dx = f(x), f(g, True)
    a, b = float((y.double() * g.double()).sum()), float((x.double() * dx.double()).sum())
    # each of the M * H * D terms is off by at most 10 steps of 1.25 (|x1| + |x2|) |g|
    assert abs(a - b) <= 2 * 10 * 2.0 ** -24 * 1.25 * 2 * float((x.abs().max() * g.abs().sum()).item())
    for at in ((0, 0), (2, 33), (3, 47), (3, 50), (3, 127)):
        e = torch.zeros_like(x)
        e[at] = 1.0
        d = ((f(x + e) - f(x - e)).double() * g.double()).sum() / 2  # linear: the step need not be small
        # the two forwards are off by 10 steps of |x| + 1 at the partner pair
        assert abs(float(d) - float(dx[at])) <= 40 * 2.0 ** -24 * 2.5 * (float(x.abs().max()) + 1) * float(g.abs().max())


def test_captured_and_other_stream(gpu):
    import e2mi
    import torch
    M, H, D = 33, 3, 256
    q = torch.randn((M, H * D), device=gpu).half()
    pos = torch.arange(M, dtype=torch.int32, device=gpu)
    freqs = e2mi.rope_freqs(D).to(gpu)
    want, _ = e2mi.rope(q, None, pos, freqs, H, 0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, _ = e2mi.rope(q, None, pos, freqs, H, 0, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        e2mi.rope(q, None, pos, freqs, H, 0, q_out=out)
    for step in range(3):
        pos += 100
        graph.replay()
        want, _ = e2mi.rope(q, None, pos, freqs, H, 0)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_feeds_the_packed_attention(gpu):
    """Next to the framework's own stage: rows that e2mi_qkv_norm_rope_packed leaves unturned (cos 1, sin 0)
    and e2mi_rope turns are those that it turns itself from tables of the same angles, up to the rounding of
    the unturned f16 rows (half a step of each of a pair's values) and of the tables."""
    import e2mi
    import torch
    M, H, KV, D = 40, 3, 1, 256
    g = torch.Generator(device=gpu).manual_seed(5)
    qkv = torch.randn((M, (H + 2 * KV) * D), generator=g, device=gpu)
    gamma = torch.ones(D, device=gpu)
    pos = torch.arange(M, dtype=torch.int32, device=gpu)
    freqs = e2mi.rope_freqs(D, 10000.0).to(gpu)
    a = torch.arange(M, device=gpu).double()[:, None] * freqs[None]
    cos, sin = (torch.cat([f(a)] * 2, 1).float().contiguous() for f in (torch.cos, torch.sin))
    want = e2mi.qkv_norm_rope_packed(qkv, pos, H, KV, gamma, gamma, cos, sin)
    flat = e2mi.qkv_norm_rope_packed(qkv, pos, H, KV, gamma, gamma, torch.ones_like(cos), torch.zeros_like(sin))
    q, k = e2mi.rope(flat[0], flat[1], pos, freqs, H, KV, q_out=flat[0], k_out=flat[1])
    for got, ref in ((q, want[3]), (k, want[4])):
        x = ref.abs().view(M, -1, D)
        pair = (x[..., :D // 2] + x[..., D // 2:]).repeat(1, 1, 2).view_as(ref) * 2 ** 0.5
        assert bool(((got.float() - ref).abs() <= 2.0 ** -11 * (pair + ref.abs()) + 2.0 ** -20 + 2.0 ** -24).all())
