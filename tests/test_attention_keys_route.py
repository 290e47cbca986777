"""Which kernel and how many shares the attention over keys takes (keys_route_*, attn_keys.hip; host functions, 256 CUs): the
rules' two sides."""
import ctypes as C

import pytest


def _plan(name, *a):
    import e2mi
    out = (C.c_int * 6)()
    getattr(e2mi.load(), name)(*a, out)
    return list(out)


def prefix(Mq, Mk, P, B, max_q, max_k, H, KV, D):
    return _plan("_ZN4e2mi17keys_route_prefixEiiiiiiiiiPi", Mq, Mk, P, B, max_q, max_k, H, KV, D)


def blocks(Mk, B, max_q, H, KV, D, q_block, n_sel):
    return _plan("_ZN4e2mi17keys_route_blocksEiiiiiiiiiPi", B * max_q, Mk, B, max_q, H, KV, D, q_block, n_sel)


def test_shares_fill_rounds():
    """Shares by what a call takes: a round of workgroups that is begun is paid for."""
    assert prefix(1500, 1500, 4096, 1, 1500, 1500, 4, 1, 512)[3:5] == [4, 5]     # 47 row tiles: 235 workgroups, one a CU
    assert prefix(40, 40 * 8192, 8, 40, 1, 8192, 8, 4, 256)[3:5] == [0, 3]       # 160: 480, two rounds
    assert prefix(1, 0, 531, 1, 1, 0, 3, 1, 256)[3:5] == [0, 1]                  # a short walk in one launch
    assert prefix(1, 0, 531, 1, 1, 0, 3, 1, 512)[4] > 1
    assert prefix(1, 0, 8192, 1, 1, 0, 4, 1, 256)[4] >= 32
    assert prefix(8, 8 * 64, 16384, 8, 1, 64, 4, 1, 256)[3:5] == [0, 32]         # of a shared prefix in multiples of 8
    for D in (64, 128, 256, 512):
        for B in (1, 7, 300):
            for n in (1, 90, 2000):
                p = prefix(B * n, B * n, 5000, B, n, n, 4, 2, D)
                assert 1 <= p[4] and p[2] + p[4] <= 128, p


# (Mq, Mk, P, B, max_q, max_k, H, KV, D) -> apart, the prefix's nw, own nw
@pytest.mark.parametrize("shape,apart,pre,own", [
    ((1, 24, 512, 1, 1, 19, 3, 1, 256), 0, None, 0),
    ((64, 4096, 2048, 64, 1, 64, 4, 1, 256), 0, None, 0),       # 64 tokens behind 2048 keys: each reads them
    ((64, 4096, 16384, 64, 1, 64, 4, 1, 256), 1, 0, 0),         # behind 16384: shared
    ((256, 16384, 16384, 256, 1, 64, 4, 2, 256), 1, 4, 0),
    ((512, 4096, 2048, 64, 8, 64, 4, 1, 256), 0, None, 0),
    ((64 * 512, 64 * 512, 2048, 64, 512, 512, 3, 1, 256), 0, None, 4),
    ((64 * 512, 64 * 512, 200000, 64, 512, 512, 3, 1, 256), 0, None, 4),  # long sequences never share a prefix's tiles
    ((128, 0, 4096, 1, 128, 0, 4, 1, 256), 0, None, 0),
    ((128, 0, 4096, 1, 128, 0, 4, 1, 512), 0, None, 2),
    ((64, 0, 4096, 1, 64, 0, 4, 1, 512), 0, None, 0),
])
def test_prefix(shape, apart, pre, own):
    p = prefix(*shape)
    assert p[0] == apart and p[3] == own and (pre is None or p[1] == pre), p
    assert 1 <= p[4] and p[2] + p[4] <= 128


@pytest.mark.parametrize("shape,nw", [
    ((8192, 1, 8192, 4, 1, 256, 8, 16), 2), ((8192, 1, 8192, 4, 1, 256, 4, 16), 0), ((8192, 1, 8192, 4, 1, 512, 4, 16), 0), ((8192, 1, 8192, 4, 1, 512, 6, 16), 2),
    ((8192, 1, 2048, 4, 1, 128, 8, 16), 0), ((8192, 1, 8192, 4, 1, 128, 8, 16), 2), ((16384, 1, 16384, 3, 1, 256, 32, 16), 3),
    ((65536, 16, 1, 4, 1, 256, 1, 32), 0), ((16384, 1, 16384, 4, 1, 256, 64, 16), 4),
])
def test_blocks(shape, nw):
    assert blocks(*shape)[3] == nw
