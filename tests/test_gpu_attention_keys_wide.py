"""The kernel for many rows (k_keys_wide) behind e2mi_attention_prefix and e2mi_attention_blocks: every head dim, number of row
groups, type, and way of sharing, at sizes whose plan is asked first; against softmax in 64 bits."""
import numpy as np
import pytest

from keys_util import MARK, check, make, reference, route_blocks, route_prefix

pytestmark = pytest.mark.gpu


def _run(c, scale, causal=False, **over):
    import e2mi
    a = dict(k_start=c["k_start"], k_len=c["k_len"], max_k=c["max_k"], scale=scale, causal=causal, ctx=c["ctx"])
    a.update(over)
    return e2mi.attention_prefix(c["q"], c["k"], c["vt"], c["pk"], c["pvt"], c["q_start"], c["q_len"], c["max_q"], c["H"], c["KV"], **a)


def _lens(seed, n, lo, hi):
    r = np.random.default_rng(seed)
    return [hi] + [int(v) for v in r.integers(lo, hi + 1, n - 1)]


PREFIX = [
    # dtype, H, KV, D, q lengths, k lengths (None: the q's), prefix, the plan's nw (own launch)
    ("float16", 4, 1, 256, _lens(1, 3, 300, 701), None, 1333, 4),         # odd prefix: V^T copied
    ("bfloat16", 3, 1, 256, _lens(2, 120, 9, 21), None, 2048, 2),         # 63 rows: two row groups
    ("bfloat16", 3, 1, 256, _lens(3, 70, 0, 32), _lens(4, 70, 0, 90), 2100, 3),   # 96 rows, some without any
    ("bfloat16", 3, 1, 256, _lens(3, 70, 0, 32), _lens(4, 70, 0, 90), 1100, 0),   # the other kernel, at its largest
    ("float16", 8, 2, 128, _lens(5, 4, 500, 1500), None, 256, 4),
    ("bfloat16", 4, 1, 128, _lens(6, 400, 1, 16), _lens(7, 400, 0, 40), 1000, 2),
    ("float16", 6, 1, 128, _lens(8, 300, 3, 16), None, 1001, 3),
    ("float16", 8, 1, 64, _lens(9, 2, 2600, 3100), _lens(10, 2, 33, 70), 500, 4),
    ("bfloat16", 4, 1, 64, _lens(11, 700, 5, 16), _lens(12, 700, 8, 9), 1200, 2),
    ("float16", 6, 1, 64, _lens(13, 500, 5, 16), None, 1200, 3),
    ("float16", 4, 1, 512, _lens(14, 2, 100, 301), None, 777, 2),         # the key range in shares
    ("bfloat16", 8, 2, 512, _lens(15, 2, 64, 70), _lens(16, 2, 500, 900), 1030, 2),
    ("float16", 3, 1, 512, _lens(17, 30, 1, 21), None, 1001, 2),
    ("bfloat16", 4, 1, 512, _lens(18, 30, 12, 24), None, 600, 2),
    ("bfloat16", 3, 1, 512, _lens(25, 90, 25, 31), None, 1001, 3),
    ("float16", 4, 1, 512, _lens(26, 3, 900, 1201), None, 555, 4),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", PREFIX, ids=lambda c: "-".join(map(str, c[:4])) + f"-q{max(c[4])}x{len(c[4])}-p{c[6]}")
def test_prefix(gpu, case, causal):
    dtype, H, KV, D, ql, kl, P, nw = case
    c = make(gpu, 31, dtype, H, KV, D, ql, kl, P)
    assert route_prefix(c)[:4:3] == [0, nw], route_prefix(c)
    scale = D ** -0.5
    check(c, _run(c, scale, causal), *reference(c, scale, causal))


@pytest.mark.parametrize("dtype,H,KV,D,B,P,pre,own", [
    ("bfloat16", 4, 2, 256, 300, 6000, 0, 0), ("bfloat16", 4, 2, 256, 300, 20000, 4, 0), ("float16", 4, 1, 128, 300, 9001, 4, 0), ("float16", 4, 1, 128, 300, 60001, 4, 0),
    ("float16", 8, 1, 64, 300, 16001, 4, 0), ("bfloat16", 4, 2, 512, 130, 3000, 2, 0)])
def test_tokens_of_many_streams(gpu, dtype, H, KV, D, B, P, pre, own):
    """The prefix by the rows of all streams, their own keys by stream, each in the kernel its rule names, joined."""
    c = make(gpu, 32, dtype, H, KV, D, [1] * B, _lens(19, B, 0, 200), P)
    plan = route_prefix(c)
    assert plan[:2] + plan[3:4] == [1, pre, own] and plan[2] > 1, plan
    check(c, _run(c, D ** -0.5), *reference(c, D ** -0.5, False))


BLOCKS = [
    # dtype, H, KV, D, q lengths, k lengths (None: the q's), q_block, n_sel, nw
    ("float16", 3, 1, 256, [4500], None, 32, 12, 3),
    ("bfloat16", 4, 2, 256, _lens(20, 4, 60, 2900), None, 16, 14, 2),
    ("float16", 4, 1, 256, [3333], None, 64, 7, 0),
    ("float16", 4, 1, 256, [5555], None, 64, 11, 4),                      # 256 rows: two tiles of 128
    ("bfloat16", 4, 1, 128, _lens(21, 70, 1, 300), None, 24, 4, 3),       # more than 64 sequences
    ("float16", 16, 4, 128, _lens(22, 3, 500, 2600), None, 16, 9, 2),
    ("float16", 8, 1, 64, [8200], _lens(23, 1, 700, 700), 16, 6, 4),
    ("float16", 4, 1, 512, [1500, 31], None, 16, 8, 2),
    ("bfloat16", 4, 1, 512, [1111], None, 33, 12, 2),
    ("float16", 4, 1, 512, [3000, 2000, 7], None, 33, 20, 4),             # 132 rows: a tile of 128, one of 4
    ("bfloat16", 4, 1, 512, [3000, 2000, 7], None, 24, 20, 3),
    ("float16", 4, 1, 512, [640], [2000], 4, 6, 0),                       # 16 rows a list
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", BLOCKS, ids=lambda c: "-".join(map(str, c[:4])) + f"-q{max(c[4])}x{len(c[4])}-b{c[6]}-n{c[7]}")
def test_blocks(gpu, case, causal):
    import e2mi
    dtype, H, KV, D, ql, kl, qb, n_sel, nw = case
    c = make(gpu, 33, dtype, H, KV, D, ql, kl)
    assert route_blocks(c, qb, n_sel)[3] == nw, route_blocks(c, qb, n_sel)
    bounds = e2mi.block_bounds(c["k"], c["k_start"], c["k_len"], c["max_k"], KV)
    sel = e2mi.block_select(c["q"], bounds, c["q_start"], c["q_len"], c["k_len"], c["max_q"], c["max_k"], H, KV, qb, n_sel, n_local=1,
                            n_first=1, causal=causal)
    s = sel.cpu().numpy()

    def keys(b, i, a):
        blocks = s[b, i, a]
        return (64 * blocks[blocks >= 0][:, None] + np.arange(64)).ravel()

    got = e2mi.attention_blocks(c["q"], c["k"], c["vt"], sel, c["q_start"], c["q_len"], c["k_start"], c["k_len"], c["max_q"], c["max_k"], H,
                                KV, qb, scale=D ** -0.5, causal=causal, ctx=c["ctx"])
    check(c, got, *reference(c, D ** -0.5, causal, keys, qb))


def test_quantized_pair(gpu):
    """Within half a step of each 128-dim scale of the context, rows outside the sequences zero; plain and in shares."""
    for dtype, H, KV, D, ql, P in (("float16", 4, 1, 256, _lens(1, 3, 300, 701), 1333), ("bfloat16", 4, 2, 128, [900, 3000], 400),
                                   ("float16", 4, 1, 512, [301, 100], 777)):
        c = make(gpu, 34, dtype, H, KV, D, ql, None, P)
        assert route_prefix(c)[3] >= 2
        y, tol = reference(c, D ** -0.5, False)
        cq, cs = _run(c, D ** -0.5, ctx=None, quant=True)
        live = c["liveq"].cpu().numpy()
        s = np.repeat(cs.cpu().numpy().astype(np.float64), 128, 1)
        off = np.abs(cq.cpu().numpy() * s - y)
        assert np.all((off <= tol + s * 0.5 * (1 + 2.0 ** -20))[live])
        assert int(cq[~c["liveq"]].abs().max()) == 0


def test_replayed_with_other_lengths(gpu):
    import torch
    ql = _lens(1, 3, 300, 701)
    c = make(gpu, 35, "float16", 4, 1, 256, ql, None, 1333)
    assert route_prefix(c)[3] == 4
    _run(c, 0.0625)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run(c, 0.0625)
    for lens in (ql, [700, 0, 1], [5, 300, 33]):
        lens = [min(n, f) for n, f in zip(lens, ql)]
        c["q_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["k_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        for s, n, f in zip(c["qs"], lens, ql):
            c["liveq"][s:s + f] = False
            c["liveq"][s:s + n] = True
        c["q_lens"], c["k_lens"] = lens, lens
        c["ctx"].fill_(MARK)
        graph.replay()
        got = c["ctx"].clone()
        c["ctx"].fill_(MARK)
        eager = _run(c, 0.0625)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        check(c, got, *reference(c, 0.0625, False))


def test_sharp_softmax_and_repeats(gpu):
    """Logits hundreds apart in this kernel, and the same bits on a second run."""
    import torch
    c = make(gpu, 36, "float16", 3, 1, 256, _lens(24, 3, 500, 901), None, 512, spread=6.0)
    assert route_prefix(c)[3] == 4
    got = _run(c, 1.0).clone()
    check(c, got, *reference(c, 1.0, False))
    assert torch.equal(got, _run(c, 1.0))


def test_caches_past_the_wide_kernels_offsets(gpu):
    """V^T of a pitch past 2^23 columns: many rows take the kernel for few."""
    import torch
    cols = (1 << 23) + 8
    c = make(gpu, 37, "bfloat16", 4, 1, 64, [2000], [2000], 0)
    y, tol = reference(c, 0.125, True)
    vt = torch.zeros((1, 64, cols), dtype=torch.bfloat16, device=gpu)
    k0 = cols - 2008
    vt[:, :, k0:k0 + 2000] = c["vt"][:, :, c["ks"][0]:c["ks"][0] + 2000]
    k = torch.zeros((cols, 64), dtype=torch.bfloat16, device=gpu)
    k[k0:k0 + 2000] = c["k"][c["ks"][0]:c["ks"][0] + 2000]
    c["k"], c["vt"], c["k_start"] = k, vt, torch.tensor([k0], dtype=torch.int32, device=gpu)
    check(c, _run(c, 0.125, True), y, tol)


def test_context_and_pair_at_once(gpu):
    """Both outputs of one call are those of two calls, in this kernel, in shares, and in the kernel for few rows."""
    import ctypes as C
    import e2mi
    import torch
    for D, ql, P, nw in ((256, _lens(1, 3, 300, 701), 1333, 4), (512, [301, 100], 777, 2), (128, [40, 3], 30, 0)):
        c = make(gpu, 38, "float16", 4, 1, D, ql, None, P)
        plan = route_prefix(c)
        assert plan[3] == nw
        ctx = _run(c, D ** -0.5).clone()
        cq, cs = _run(c, D ** -0.5, ctx=None, quant=True)
        got, gq, gs = torch.full_like(ctx, MARK), torch.zeros_like(cq), torch.zeros_like(cs)
        lib, Mk, ldv = e2mi.load(), c["k"].shape[0], c["vt"].stride(1)
        need = lib.e2mi_attention_prefix_workspace_bytes(c["Mq"], Mk, ldv, P, P, len(ql), c["max_q"], c["max_k"], 4, 1, D)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu)
        p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        e2mi.check(lib.e2mi_attention_prefix(
            torch.cuda.current_stream().cuda_stream, 0, p(c["q"]), 4 * D, c["Mq"], p(c["k"]), D, p(c["vt"]), ldv, Mk, p(c["pk"]), D,
            p(c["pvt"]), P, P, p(c["q_start"]), p(c["q_len"]), p(c["k_start"]), p(c["k_len"]), len(ql), c["max_q"], c["max_k"], 4, 1, D,
            D ** -0.5, 0, p(got), 4 * D, p(gq), p(gs), p(ws), need), "attention_prefix")
        assert torch.equal(got, ctx) and torch.equal(gq, cq) and torch.equal(gs, cs)


def test_empty_batches(gpu):
    """No rows or no sequences: empty results; lists of sequences without rows: none."""
    import e2mi
    import torch
    none, i32 = torch.empty(0, 512, dtype=torch.float16, device=gpu), lambda n: torch.zeros(n, dtype=torch.int32, device=gpu)  # noqa: E731
    k, vt, some = torch.zeros(64, 256, dtype=torch.float16, device=gpu), torch.zeros(1, 256, 64, dtype=torch.float16, device=gpu), i32(2)
    assert e2mi.attention_prefix(none, None, None, k, vt, some, some, 4, 2, 1).shape == (0, 512)
    assert int(e2mi.attention_prefix(k, None, None, k, vt, i32(0), i32(0), 4, 1, 1).abs().max()) == 0
    assert e2mi.rope(none, None, i32(0), torch.ones(128, dtype=torch.float64, device=gpu), 2, 0)[0].shape == (0, 512)
    bounds = e2mi.block_bounds(k, some, some + 64, 64, 1)
    sel = e2mi.block_select(none, bounds, some, some, some + 64, 4, 64, 2, 1, 4, 3)
    assert sel.shape == (2, 1, 1, 3) and int(sel.max()) == -1 == int(sel.min())
    assert e2mi.attention_blocks(none, k, vt, sel, some, some, some, some + 64, 4, 64, 2, 1, 4).shape == (0, 512)
