"""Refusals of the attention over a shared prefix and over selected blocks, and of the selection itself: every
one before a launch, so no GPU is needed and no address is read."""
import pytest

X = 1 << 20
PREFIX = dict(stream=None, dtype=0, q=X, ldq=768, Mq=64, k=2 * X, ldk=256, vt=3 * X, ldv=64, Mk=64, pk=4 * X, ldpk=256, pvt=5 * X,
              ldpv=33, P=33, qs=6 * X, ql=7 * X, ks=8 * X, kl=9 * X, B=2, max_q=32, max_k=32, H=3, KV=1, D=256, scale=0.0625, causal=0,
              ctx=10 * X, ldc=768, cq=None, cs=None, ws=11 * X, wn=1 << 40)
BLOCKS = dict(stream=None, dtype=0, q=X, ldq=768, Mq=64, k=2 * X, ldk=256, vt=3 * X, ldv=64, Mk=64, qs=6 * X, ql=7 * X, ks=8 * X, kl=9 * X,
              B=2, max_q=32, max_k=32, H=3, KV=1, D=256, q_block=16, sel=12 * X, n_sel=4, scale=0.0625, causal=0, ctx=10 * X, ldc=768,
              cq=None, cs=None, ws=11 * X, wn=1 << 40)
BOUNDS = dict(stream=None, dtype=0, k=2 * X, ldk=256, Mk=64, ks=8 * X, kl=9 * X, B=2, max_k=64, KV=1, D=256, bounds=3 * X, scale=4 * X)
SELECT = dict(stream=None, dtype=0, q=X, ldq=768, Mq=64, bounds=2 * X, scale=3 * X, qs=6 * X, ql=7 * X, kl=9 * X, B=2, max_q=32, max_k=640,
              H=3, KV=1, D=256, q_block=16, n_sel=4, n_first=1, n_local=1, causal=0, sel=12 * X, ws=11 * X, wn=1 << 40)
NOTHING = dict(B=0)  # what is checked, and then has nothing to do

ROWS = [dict(dtype=2), dict(dtype=-1), dict(Mq=-1), dict(B=-1), dict(B=65536), dict(max_q=-1), dict(max_k=-1), dict(H=0), dict(KV=0),
        dict(KV=2), dict(D=96), dict(D=0), dict(q=None), dict(q=X + 8), dict(ldq=767), dict(ldq=772), dict(ldq=1 << 40), dict(qs=None),
        dict(ql=None), dict(kl=None)]
KEYS = [dict(k=None), dict(k=2 * X + 2), dict(ldk=255), dict(ldk=260), dict(vt=None), dict(vt=3 * X + 1), dict(vt=3 * X + 2), dict(ldv=63), dict(ldv=1 << 26), dict(ldk=1 << 24), dict(Mk=-1),
        dict(ks=None)]
OUT = [dict(ctx=None), dict(ctx=10 * X + 4), dict(ldc=760), dict(ldc=770), dict(cq=X), dict(cs=X), dict(ctx=None, cq=X), dict(cq=X + 4, cs=X),
       dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan"))]


def _refused(fn, name, base, over):
    import e2mi
    lib = e2mi.load()
    assert getattr(lib, fn)(*{**base, **over}.values()) == -1, over
    assert name in e2mi.last_error(), (over, e2mi.last_error())


@pytest.mark.parametrize("over", ROWS + KEYS + OUT + [dict(P=-1), dict(pk=None), dict(pvt=None), dict(ldpv=32), dict(ldpk=8)], ids=str)
def test_prefix(over):
    _refused("e2mi_attention_prefix", "attention_prefix", PREFIX, over)
    if "B" not in over:
        _refused("e2mi_attention_prefix", "attention_prefix", {**PREFIX, **NOTHING}, over)


@pytest.mark.parametrize("over", ROWS + KEYS + OUT + [dict(sel=None), dict(q_block=0), dict(q_block=1025), dict(n_sel=0), dict(n_sel=2049)],
                         ids=str)
def test_blocks(over):
    _refused("e2mi_attention_blocks", "attention_blocks", BLOCKS, over)


@pytest.mark.parametrize("over", [dict(dtype=2), dict(D=96), dict(KV=0), dict(B=-1), dict(B=65536), dict(max_k=-1), dict(Mk=-1), dict(k=None),
                                  dict(k=X + 2), dict(ldk=200), dict(ldk=257), dict(ks=None), dict(kl=None), dict(bounds=None),
                                  dict(bounds=X + 8), dict(scale=None)], ids=str)
def test_bounds(over):
    _refused("e2mi_block_bounds", "block_bounds", BOUNDS, over)


@pytest.mark.parametrize("over", [o for o in ROWS] + [dict(max_k=(1 << 21) + 1), dict(q_block=0), dict(q_block=1025), dict(n_sel=0),
                                                      dict(n_sel=2049), dict(n_first=-1), dict(n_local=-1), dict(n_first=3),
                                                      dict(n_local=3), dict(sel=None), dict(bounds=None), dict(scale=None),
                                                      dict(ws=None), dict(wn=8)], ids=str)
def test_select(over):
    _refused("e2mi_block_select", "block_select", SELECT, over)


def test_nothing_to_do_succeeds():
    import e2mi
    lib = e2mi.load()
    for over in (dict(B=0), dict(Mq=0), dict(max_q=0)):
        assert lib.e2mi_attention_prefix(*{**PREFIX, **over}.values()) == 0
        assert lib.e2mi_attention_blocks(*{**BLOCKS, **over}.values()) == 0
    for over in (dict(B=0), dict(Mk=0), dict(max_k=0)):
        assert lib.e2mi_block_bounds(*{**BOUNDS, **over}.values()) == 0
    for over in (dict(B=0), dict(max_q=0)):
        assert lib.e2mi_block_select(*{**SELECT, **over}.values()) == 0


def test_workspace_sizes():
    """Zero for what is refused; enough for every share of a few tokens; too small a workspace is refused."""
    import e2mi
    lib = e2mi.load()
    size = lib.e2mi_attention_prefix_workspace_bytes
    assert size(64, 64, 64, 33, 33, 2, 32, 32, 3, 1, 96) == 0 and size(64, 64, 64, -1, 33, 2, 32, 32, 3, 1, 256) == 0
    assert lib.e2mi_attention_blocks_workspace_bytes(64, 64, 64, 2, 32, 3, 1, 256, 0, 4) == 0
    assert lib.e2mi_block_select_workspace_bytes(2, 32, 640, 1, 16) == 2 * 2 * 10 * 4
    few = dict(PREFIX, Mq=1, B=1, max_q=1, P=4096, ldpv=4096)
    need = size(1, 64, 64, 4096, 4096, 1, 1, 32, 3, 1, 256)
    assert need >= 2 * 3 * (256 + 2) * 4
    for over in (dict(ws=None, wn=0), dict(wn=need - 1), dict(ws=X + 4)):
        assert lib.e2mi_attention_prefix(*{**few, **over}.values()) == -1
        assert "workspace" in e2mi.last_error()


def test_wrapper_refusals_need_no_gpu():
    import e2mi
    import torch
    x, i = torch.zeros(8, 512, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    for H, KV in ((0, 1), (2, 0), (-2, 1), (3, 1)):
        with pytest.raises(e2mi.E2MIError, match="attention_prefix"):
            e2mi.attention_prefix(x, None, None, None, None, i, i, 8, H, KV)
        with pytest.raises(e2mi.E2MIError, match="attention_blocks"):
            e2mi.attention_blocks(x, x, x, i, i, i, i, i, 8, 8, H, KV, 4)
        with pytest.raises(e2mi.E2MIError, match="block_select"):
            e2mi.block_select(x, (x, x), i, i, i, 8, 8, H, KV, 4, 2)
    with pytest.raises(e2mi.E2MIError, match="block_bounds"):
        e2mi.block_bounds(x, i, i, 8, 0)
