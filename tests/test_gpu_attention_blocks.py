"""Selected key blocks: bounds and selection exactly against whole numbers in 64 bits, the attention over lists
against softmax in 64 bits, and the three together after e2mi_rope."""
import numpy as np
import pytest

from keys_util import MARK, check, make, reference

pytestmark = pytest.mark.gpu
BLOCK = 64
INV127 = np.float32(np.uint32(0x3c010204).view(np.float32))


def quantized(x):
    """Rows of x (32-bit values) by the framework's quantizer: bytes and scale."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(-1, keepdims=True)
    one = np.ones_like(amax)
    inv = np.where(amax > 0, np.float32(127) / np.where(amax > 0, amax, one), one).astype(np.float32)
    sc = np.where(amax > 0, amax * INV127, one).astype(np.float32)
    return np.clip(np.rint((x * inv).astype(np.float32)), -128, 127).astype(np.int64), sc[..., 0]


def _f32(t):
    return t.float().cpu().numpy()


def bounds_of(c):
    KV, D = c["KV"], c["D"]
    NB = -(-c["max_k"] // BLOCK)
    k = _f32(c["k"])
    out = np.zeros((len(c["k_lens"]), NB, KV, 2 * D), np.int64)
    sc = np.zeros(out.shape[:3], np.float32)
    for b, (k0, nk) in enumerate(zip(c["ks"], c["k_lens"])):
        for n in range(-(-nk // BLOCK)):
            rows = k[k0 + n * BLOCK:k0 + min(nk, (n + 1) * BLOCK)].reshape(-1, KV, D)
            out[b, n], sc[b, n] = quantized(np.concatenate([rows.max(0), rows.min(0)], -1))
    return out, sc


def select_of(c, bounds, qb, n_sel, n_first=0, n_local=0, causal=False):
    """The lists by their definition: whole-number dots, two 32-bit products, a stable sort."""
    H, KV, D, G = c["H"], c["KV"], c["D"], c["H"] // c["KV"]
    NQ = -(-c["max_q"] // qb)
    q = _f32(c["q"])
    sel = np.full((len(c["q_lens"]), NQ, KV, n_sel), -1, np.int64)
    b8, bs = bounds
    for b, (q0, nq, nk) in enumerate(zip(c["qs"], c["q_lens"], c["k_lens"])):
        nb = -(-nk // BLOCK)
        for a in range(KV):
            for i in range(-(-nq // qb)):
                toks = np.arange(i * qb, min(nq, (i + 1) * qb))
                best = np.full(nb, -np.inf, np.float32)
                last = toks + nk - nq if causal else np.full(toks.size, nk - 1)
                for t, far in zip(toks, last):
                    for h in range(a * G, (a + 1) * G):
                        q8, qs = quantized(q[q0 + t, h * D:(h + 1) * D])
                        dot = np.maximum(q8 * b8[b, :nb, a, :D], q8 * b8[b, :nb, a, D:]).sum(-1)
                        s = dot.astype(np.float32) * qs
                        see = np.arange(nb) * BLOCK <= far
                        best = np.where(see, np.maximum(best, s), best)
                score = (best * bs[b, :nb, a]).astype(np.float32)
                can = np.arange(nb) * BLOCK <= last[-1]
                n = np.arange(nb)
                must = n < n_first
                if n_local:
                    lo, hi = (toks[0] + nk - nq) // BLOCK, (toks[-1] + nk - nq) // BLOCK
                    must |= (n >= lo - (n_local - 1)) & (n <= hi + (0 if causal else n_local - 1))
                score = np.where(must, np.float32(np.inf), score)[can]
                pick = np.sort(n[can][np.argsort(-score, kind="stable")[:n_sel]])
                sel[b, i, a, :pick.size] = pick
    return sel


def _bounds(c):
    import e2mi
    return e2mi.block_bounds(c["k"], c["k_start"], c["k_len"], c["max_k"], c["KV"])


def _select(c, bounds, qb, n_sel, **kw):
    import e2mi
    return e2mi.block_select(c["q"], bounds, c["q_start"], c["q_len"], c["k_len"], c["max_q"], c["max_k"], c["H"], c["KV"], qb, n_sel, **kw)


def _attend(c, sel, qb, scale, causal=False, **kw):
    import e2mi
    a = dict(scale=scale, causal=causal, ctx=c["ctx"])
    a.update(kw)
    return e2mi.attention_blocks(c["q"], c["k"], c["vt"], sel, c["q_start"], c["q_len"], c["k_start"], c["k_len"], c["max_q"], c["max_k"],
                                 c["H"], c["KV"], qb, **a)


CASES = [
    # dtype, H, KV, D, q lengths, k lengths (None: the q's), q_block, n_sel, n_first, n_local
    ("float16", 3, 1, 256, [1, 1, 1], [1000, 64, 65], 1, 6, 1, 1),        # tokens: a query block of 3 rows
    ("bfloat16", 8, 1, 128, [1, 1], [900, 1], 1, 3, 0, 0),                # 8 rows
    ("float16", 4, 2, 64, [40, 3], [700, 333], 5, 4, 1, 0),               # 10 rows: two query blocks a tile
    ("float16", 3, 1, 256, [130, 0, 70, 1], None, 16, 2, 0, 1),           # 48 rows, an empty sequence
    ("bfloat16", 4, 1, 512, [200], None, 64, 3, 1, 1),                    # 256 rows
    ("float16", 6, 2, 128, [500, 129], None, 32, 5, 1, 2),
    ("float16", 2, 2, 256, [90], [30], 16, 8, 0, 1),                      # fewer keys than queries
    ("bfloat16", 16, 4, 64, [65, 64], [640, 2000], 24, 7, 0, 0),
]


def _ids(c):
    return "-".join(map(str, c[:4])) + f"-q{max(c[4])}x{len(c[4])}-b{c[6]}-n{c[7]}"


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_selection_is_exact(gpu, case, causal):
    dtype, H, KV, D, ql, kl, qb, n_sel, n_first, n_local = case
    c = make(gpu, 21, dtype, H, KV, D, ql, kl)
    want_b = bounds_of(c)
    got_b = _bounds(c)
    for b, nk in enumerate(c["k_lens"]):
        nb = -(-nk // BLOCK)
        assert np.array_equal(got_b[0][b, :nb].cpu().numpy(), want_b[0][b, :nb])
        assert np.array_equal(got_b[1][b, :nb].cpu().numpy(), want_b[1][b, :nb])
    got = _select(c, got_b, qb, n_sel, n_first=n_first, n_local=n_local, causal=causal).cpu().numpy()
    assert np.array_equal(got, select_of(c, want_b, qb, n_sel, n_first, n_local, causal))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CASES, ids=_ids)
def test_attention_over_lists(gpu, case, causal):
    dtype, H, KV, D, ql, kl, qb, n_sel, n_first, n_local = case
    c = make(gpu, 22, dtype, H, KV, D, ql, kl)
    sel = _select(c, _bounds(c), qb, n_sel, n_first=n_first, n_local=n_local, causal=causal)
    s = sel.cpu().numpy()

    def keys(b, i, a):
        blocks = s[b, i, a]
        return [64 * n + j for n in blocks[blocks >= 0] for j in range(64)]

    check(c, _attend(c, sel, qb, D ** -0.5, causal), *reference(c, D ** -0.5, causal, keys, qb))


def test_every_block_listed_is_the_whole_attention(gpu):
    """Lists of all blocks: the same context as attention over all keys, within the tolerance of each."""
    import e2mi
    c = make(gpu, 23, "float16", 3, 1, 256, [150, 33], None)
    sel = _select(c, _bounds(c), 32, 8)
    y, tol = reference(c, 0.0625, False)
    check(c, _attend(c, sel, 32, 0.0625), y, tol)
    c["ctx"].fill_(MARK)
    check(c, e2mi.attention_prefix(c["q"], c["k"], c["vt"], None, None, c["q_start"], c["q_len"], c["max_q"], 3, 1, scale=0.0625,
                                   ctx=c["ctx"]), y, tol)


def test_lists_of_a_callers_own(gpu):
    """Any order, entries past the last block and negative ones passed over, an entry twice counted twice, an empty list."""
    import torch
    c = make(gpu, 24, "bfloat16", 4, 2, 128, [40], [300])
    sel = torch.tensor([[[[4, 0, -1, 5, 1 << 20], [2, 2, -7, 2 ** 31 - 1, -2 ** 31]],
                         [[-1] * 5, [1, 99, 0, 3, 3]]]], dtype=torch.int32, device=gpu)
    read = {(0, 0): [4, 0], (0, 1): [2, 2], (1, 0): [], (1, 1): [1, 0, 3, 3]}

    def keys(b, i, a):
        return [64 * n + j for n in read[i, a] for j in range(64)]

    check(c, _attend(c, sel, 32, 0.1), *reference(c, 0.1, False, keys, 32))


def test_ties_and_order(gpu):
    """Equal scores everywhere (one key repeated): the lowest blocks, and with negative scores too."""
    for sign in (1.0, -1.0):
        c = make(gpu, 25, "float16", 4, 1, 64, [3], [64 * 50 + 7])
        k0 = c["ks"][0]
        c["k"][k0:k0 + c["k_lens"][0]] = 0.5
        c["q"][c["qs"][0]:c["qs"][0] + 3] = sign
        got = _select(c, _bounds(c), 2, 9).cpu().numpy()
        assert np.array_equal(got[0, :, 0], np.tile(np.arange(9), (2, 1)))
        c["k"][k0 + 64 * 20] = 2.0 * sign  # one better block
        got = _select(c, _bounds(c), 2, 9).cpu().numpy()
        assert np.array_equal(got[0, :, 0], np.tile(np.r_[np.arange(8), 20], (2, 1)))


@pytest.mark.parametrize("blocks,n_sel", [(512, 512), (513, 40), (2049, 300), (8193, 2048), (20001, 17)])
def test_many_blocks(gpu, blocks, n_sel):
    """Each size class of the ranking, by given bounds: one dim holds the block's score, many of them equal."""
    import e2mi
    import torch
    D = 64
    rng = np.random.default_rng(blocks)
    level = rng.integers(-127, 128, blocks)
    b8 = torch.zeros((1, blocks, 1, 2 * D), dtype=torch.int8, device=gpu)
    b8[0, :, 0, 0] = torch.from_numpy(level.astype(np.int8)).to(gpu)
    b8[0, :, 0, D] = b8[0, :, 0, 0]
    sc = torch.ones((1, blocks, 1), device=gpu)
    q = torch.zeros((1, D), dtype=torch.float16, device=gpu)
    q[0, 0] = 1.0
    one = torch.ones(1, dtype=torch.int32, device=gpu)
    nk = blocks * 64 - 63
    got = e2mi.block_select(q, (b8, sc), one * 0, one, one * nk, 1, nk, 1, 1, 1, n_sel).cpu().numpy().ravel()
    assert np.array_equal(got, np.sort(np.argsort(-level, kind="stable")[:n_sel]))


def test_infinite_and_nan_keys_end(gpu):
    """A block whose keys hold an infinity or a NaN leaves the others' order as it is."""
    c = make(gpu, 26, "float16", 2, 1, 128, [4], [64 * 12])
    clean = _select(c, _bounds(c), 4, 12).cpu().numpy()
    assert np.array_equal(clean[0, 0, 0], np.arange(12))
    few = _select(c, _bounds(c), 4, 5).cpu().numpy()[0, 0, 0]
    spare = [n for n in range(12) if n not in few]
    c["k"][c["ks"][0] + 64 * spare[0] + 3, 5] = float("nan")
    got = _select(c, _bounds(c), 4, 5).cpu().numpy()[0, 0, 0]
    assert np.array_equal(got, few)
    c["k"][c["ks"][0] + 64 * spare[0] + 3, 5] = float("inf")
    got = _select(c, _bounds(c), 4, 6).cpu().numpy()[0, 0, 0]
    assert len(set(got)) == 6 and min(got) >= 0 and max(got) < 12


def test_together_after_rope(gpu):
    """As a long text goes through them: rows turned, bounds, selection, attention, in one captured graph whose lengths
    change between replays; against the 64-bit reference over the lists it chose."""
    import e2mi
    import torch
    H, KV, D, qb, n_sel = 4, 2, 128, 16, 4
    c = make(gpu, 27, "bfloat16", H, KV, D, [300, 77], None)
    pos = torch.arange(c["Mq"], dtype=torch.int32, device=gpu)
    freqs = e2mi.rope_freqs(64, 10000.0, "parts", 8.0, trained_len=2048).to(gpu)
    q0, k0 = c["q"].clone(), c["k"].clone()
    kpos = torch.arange(k0.shape[0], dtype=torch.int32, device=gpu)

    def layer():
        e2mi.rope(q0, None, pos, freqs, H, 0, layout="interleaved", q_out=c["q"])
        e2mi.rope(None, k0, kpos, freqs, 0, KV, layout="interleaved", k_out=c["k"])
        sel = _select(c, _bounds(c), qb, n_sel, n_first=1, n_local=1, causal=True)
        _attend(c, sel, qb, D ** -0.5, True)
        return sel

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sel = layer()
    full = list(c["q_lens"])
    for lens in (full, [150, 60], [299, 1]):
        c["q_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["k_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["q_lens"], c["k_lens"] = lens, lens
        for s, n, f in zip(c["qs"], lens, full):
            c["liveq"][s:s + f] = False
            c["liveq"][s:s + n] = True
        c["ctx"].fill_(MARK)
        graph.replay()
        torch.cuda.synchronize()
        got, lists = c["ctx"].clone(), sel.cpu().numpy()
        c["ctx"].fill_(MARK)
        eager = layer()
        torch.cuda.synchronize()
        assert torch.equal(got, c["ctx"]) and np.array_equal(lists, eager.cpu().numpy())
        assert np.array_equal(lists, select_of(c, bounds_of(c), qb, n_sel, 1, 1, True))

        def keys(b, i, a):
            blocks = lists[b, i, a]
            return [64 * n + j for n in blocks[blocks >= 0] for j in range(64)]

        check(c, got, *reference(c, D ** -0.5, True, keys, qb))


def test_a_prefix_turned_once(gpu):
    """Rope and the shared prefix together: keys turned at their places before the suffixes, beside the whole thing in one
    sequence's attention."""
    import e2mi
    import torch
    H, KV, D, P, n = 3, 1, 256, 100, 40
    c = make(gpu, 28, "float16", H, KV, D, [n, n], None, P)
    freqs = e2mi.rope_freqs(D, 10000.0).to(gpu)
    place = torch.zeros(c["k"].shape[0], dtype=torch.int32, device=gpu)
    for s in c["ks"]:
        place[s:s + n] = P + torch.arange(n, dtype=torch.int32, device=gpu)
    c["q"], _ = e2mi.rope(c["q"], None, place[:c["Mq"]].contiguous(), freqs, H, 0)
    _, c["k"] = e2mi.rope(None, c["k"], place, freqs, 0, KV)
    _, c["pk"] = e2mi.rope(None, c["pk"], torch.arange(P, dtype=torch.int32, device=gpu), freqs, 0, KV)
    y, tol = reference(c, 0.0625, True)
    got = e2mi.attention_prefix(c["q"], c["k"], c["vt"], c["pk"], c["pvt"], c["q_start"], c["q_len"], n, H, KV, scale=0.0625, causal=True,
                                ctx=c["ctx"])
    check(c, got, y, tol)
