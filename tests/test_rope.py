"""Rotary positions: the frequency helper against its formulas in 64 bits, and the refusals of
e2mi_rope / e2mi_rope_freqs (no GPU: every refusal comes before a launch)."""
import ctypes as C
import math

import numpy as np
import pytest


@pytest.mark.parametrize("rot", [2, 6, 64, 130, 256, 512])
@pytest.mark.parametrize("scaling", ["plain", "linear", "base", "parts"])
def test_frequencies(rot, scaling):
    import e2mi
    if scaling == "base" and rot == 2:
        with pytest.raises(e2mi.E2MIError, match="one pair"):
            e2mi.rope_freqs(rot, 10000.0, scaling, 4.0)
        return
    got = e2mi.rope_freqs(rot, 10000.0, scaling, 4.0, trained_len=4096, turns=(1.0, 32.0)).numpy()
    i = np.arange(rot // 2, dtype=np.longdouble)
    theta = np.longdouble(10000.0)
    if scaling == "base":
        theta = theta * np.longdouble(4.0) ** (np.longdouble(rot) / (rot - 2))
    f = theta ** (-2 * i / rot)
    if scaling == "linear":
        f = f / 4
    elif scaling == "parts":
        turns = 4096 * f / (2 * np.longdouble(math.pi))
        keep = np.clip((turns - 1) / 31, 0, 1)
        f = f * keep + f / 4 * (1 - keep)
    # two pow calls of at most an ulp each, the exponent's rounding times |ln f| < 16, and a few products
    assert np.all(np.abs(got - f) <= 64 * 2.0 ** -53 * f)


def test_frequency_refusals():
    import e2mi
    lib = e2mi.load()
    f = np.zeros(64)
    p = f.ctypes.data_as(C.c_void_p)
    ok = (p, 128, 1e4, 3, 4.0, 4096, 1.0, 32.0)
    assert lib.e2mi_rope_freqs(*ok) == 0
    bad = [(0, None), (1, 0), (1, -2), (1, 7), (2, 0.0), (2, float("inf")), (2, float("nan")), (3, -1), (3, 4), (4, 0.0),
           (4, float("nan")), (5, 0), (6, -1.0), (7, 1.0), (7, float("inf")), (6, float("nan"))]
    for at, v in bad:
        a = list(ok)
        a[at] = v
        assert lib.e2mi_rope_freqs(*a) == -1, (at, v)
        assert "rope_freqs" in e2mi.last_error()


def test_rope_refusals():
    import e2mi
    lib = e2mi.load()
    x = 1 << 20  # addresses are only compared: nothing here is read
    ok = dict(stream=None, dtype=0, layout=0, inverse=0, q=x, ldq=1024, qo=2 * x, ldqo=1024, H=4, k=3 * x, ldk=512, ko=4 * x,
              ldko=512, KV=2, M=8, D=256, pos=5 * x, freqs=6 * x, rot=256, mag=1.0)

    def call(**over):
        return lib.e2mi_rope(*{**ok, **over}.values())

    assert call(M=0) == 0  # nothing to do, checked like any other call
    for over in (dict(dtype=3), dict(dtype=-1), dict(layout=2), dict(M=-1), dict(D=0), dict(H=-1), dict(H=0, KV=0),
                 dict(rot=0), dict(rot=255), dict(rot=258), dict(mag=float("inf")), dict(mag=float("nan")), dict(q=None),
                 dict(qo=None), dict(k=None), dict(ko=None), dict(pos=None), dict(freqs=None), dict(ldq=1023), dict(ldko=511),
                 dict(q=x + 1), dict(freqs=6 * x + 4), dict(pos=5 * x + 2), dict(ldq=1 << 40)):
        assert call(**over) == -1, over
        assert "rope" in e2mi.last_error(), over
        assert call(**{"M": 0, **over}) == -1, over
    # overlaps: another pitch over the same rows, a shifted output, an output over the other operand
    for over in (dict(qo=x, ldqo=1032), dict(qo=x + 512), dict(qo=3 * x), dict(ko=x), dict(qo=4 * x)):
        assert call(**over) == -1, over
        assert "overlap" in e2mi.last_error(), over


def test_wrapper_refusals_need_no_gpu():
    import e2mi
    import torch
    with pytest.raises(e2mi.E2MIError, match="needs q or k"):
        e2mi.rope(None, None, None, None, 1, 1)
    x = torch.zeros(2, 256, dtype=torch.float16)
    for H, layout in ((0, "half"), (-1, "half"), (3, "half"), (1, "both")):
        with pytest.raises(e2mi.E2MIError, match="rope"):
            e2mi.rope(x, None, None, None, H, 0, layout)
    with pytest.raises(e2mi.E2MIError, match="scaling"):
        e2mi.rope_freqs(64, scaling="other")
    if not torch.cuda.is_available():
        return
    x = torch.zeros(2, 256, dtype=torch.float16)
    with pytest.raises(e2mi.E2MIError, match="current device"):
        e2mi.rope(x, None, None, None, 1, 0)
