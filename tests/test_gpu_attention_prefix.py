"""e2mi_attention_prefix against softmax in 64 bits, over lengths, masks, types and the ways it is called."""
import numpy as np
import pytest

from keys_util import MARK, check, make, reference

pytestmark = pytest.mark.gpu


def _run(c, scale, causal=False, **over):
    import e2mi
    a = dict(k_start=c["k_start"], k_len=c["k_len"], max_k=c["max_k"], scale=scale, causal=causal, ctx=c["ctx"])
    a.update(over)
    return e2mi.attention_prefix(c["q"], c["k"], c["vt"], c["pk"], c["pvt"], c["q_start"], c["q_len"], c["max_q"], c["H"], c["KV"], **a)


CASES = [
    # dtype, H, KV, D, q lengths, k lengths (None: the q's), prefix
    ("float16", 3, 1, 256, [1], [19], 512),                      # one token, shares of the range
    ("float16", 3, 1, 256, [1], [1], 1),                         # two keys in all
    ("bfloat16", 4, 2, 256, [1] * 9, [0, 1, 31, 32, 33, 64, 5, 0, 200], 700),  # tokens of many streams, some without own keys
    ("float16", 4, 4, 64, [2, 1, 3], [40, 8, 3], 33),            # no grouping, small heads
    ("float16", 3, 1, 256, [70, 0, 1, 33], None, 45),            # an empty sequence in a batch
    ("bfloat16", 4, 1, 512, [37, 130], None, 99),
    ("float16", 4, 1, 512, [1, 1], [77, 300], 1000),
    ("float16", 8, 2, 128, [129, 40, 256], None, 0),             # no prefix
    ("bfloat16", 16, 4, 128, [5, 64, 127], [60, 64, 400], 31),   # more keys than queries
    ("float16", 6, 2, 128, [40, 9], [12, 0], 0),                 # fewer keys than queries, and none at all
    ("float16", 12, 1, 64, [300], None, 130),
    ("bfloat16", 1, 1, 256, [385], [1000], 260),
]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:4])) + f"-q{max(c[4])}x{len(c[4])}-p{c[6]}")
def test_against_64_bits(gpu, case, causal):
    dtype, H, KV, D, ql, kl, P = case
    c = make(gpu, 3, dtype, H, KV, D, ql, kl, P)
    scale = D ** -0.5
    got = _run(c, scale, causal)
    check(c, got, *reference(c, scale, causal))


def test_sharp_and_flat_softmax(gpu):
    """Logits far apart (one key takes all, the running maximum moves by hundreds) and all alike."""
    for spread, scale in ((6.0, 1.0), (1.0, 1e-6)):
        c = make(gpu, 5, "float16", 3, 1, 256, [90, 1, 17], None, 150, spread=spread)
        check(c, _run(c, scale), *reference(c, scale, False))


def test_rows_that_see_nothing(gpu):
    """Causal rows before the first own key, and a sequence with no keys at all: zeros, not NaN."""
    c = make(gpu, 6, "float16", 3, 1, 256, [20, 7], [5, 0], 0)
    got = _run(c, 0.0625, True)
    y, tol = reference(c, 0.0625, True)
    check(c, got, y, tol)
    q0 = c["qs"][0]
    assert float(got[q0:q0 + 15].abs().max()) == 0.0 and float(got[c["qs"][1]:c["qs"][1] + 7].abs().max()) == 0.0
    # without own keys given at all, beside a prefix and with nothing
    import e2mi
    for pk, pvt in ((None, None), (c["k"][8:13].contiguous(), c["vt"][:, :, 8:13].contiguous())):
        out = e2mi.attention_prefix(c["q"], None, None, pk, pvt, c["q_start"], c["q_len"], c["max_q"], 3, 1, scale=0.0625)
        assert bool(torch_finite(out[c["liveq"]]))
        assert (float(out.abs().max()) == 0.0) == (pk is None)


def torch_finite(t):
    import torch
    return torch.isfinite(t).all()


def test_quantized_pair(gpu, oracle):
    """The pair for the O projection: the quantizer's bytes of the context in f32, so within half a step of it."""
    c = make(gpu, 7, "float16", 3, 1, 256, [50, 1, 9], None, 70)
    y, tol = reference(c, 0.0625, False)
    cq, cs = _run(c, 0.0625, ctx=None, quant=True)
    live = c["liveq"].cpu().numpy()
    b = cq.cpu().numpy().astype(np.float64).reshape(c["Mq"], -1, 128)
    s = cs.cpu().numpy().astype(np.float64)[..., None]
    off = np.abs((b * s).reshape(c["Mq"], -1) - y)[live]
    # half a step of the scale on top of the value's own tolerance
    lim = (tol + np.repeat(s[..., 0], 128, 1) * 0.5 * (1 + 2.0 ** -20))[live]
    assert np.all(off <= lim)
    assert int(cq[~c["liveq"]].abs().max()) == 0
    # tokens alone go through the shares' join: the same pair from there
    t = make(gpu, 8, "float16", 3, 1, 256, [1, 1], [40, 90], 600)
    y, tol = reference(t, 0.0625, False)
    cq, cs = _run(t, 0.0625, ctx=None, quant=True)
    live = t["liveq"].cpu().numpy()
    s = cs.cpu().numpy().astype(np.float64)
    off = np.abs(cq.cpu().numpy().reshape(t["Mq"], -1, 128) * s[..., None] - y.reshape(t["Mq"], -1, 128)).reshape(t["Mq"], -1)
    assert np.all(off[live] <= (tol + 0.5 * (1 + 2.0 ** -20) * np.repeat(s, 128, 1))[live])


def test_no_context_depends_on_its_batch(gpu):
    """A sequence alone, and in a batch of the same limits: the same bits (the shares of a key range follow from the
    call's sizes only)."""
    import torch
    c = make(gpu, 9, "float16", 4, 2, 256, [40, 64, 33], None, 128)
    both = _run(c, 0.0625).clone()
    again = _run(c, 0.0625)
    assert torch.equal(both, again), "two runs of one call differ"


def test_strided_rows_and_shared_ranges(gpu):
    """q as columns of a wider row buffer, k with a pitch, two sequences over the same keys, a context with a pitch."""
    import e2mi
    import torch
    c = make(gpu, 10, "bfloat16", 4, 2, 128, [33, 33], [50, 50], 40)
    c["ks"] = [c["ks"][0]] * 2  # both read the first one's keys
    c["k_start"] = torch.tensor(c["ks"], dtype=torch.int32, device=gpu)
    y, tol = reference(c, 0.1, False)
    wide_q = torch.full((c["Mq"], 4 * 128 + 24), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide_q[:, 8:8 + 512] = c["q"]
    wide_k = torch.full((c["k"].shape[0], 2 * 128 + 8), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide_k[:, :256] = c["k"]
    wide_o = torch.full((c["Mq"], 4 * 128 + 16), MARK, dtype=torch.bfloat16, device=gpu)
    e2mi.attention_prefix(wide_q[:, 8:520], wide_k[:, :256], c["vt"], c["pk"], c["pvt"], c["q_start"], c["q_len"], c["max_q"], 4, 2,
                          k_start=c["k_start"], k_len=c["k_len"], max_k=c["max_k"], scale=0.1, ctx=wide_o[:, 8:520])
    check(c, wide_o[:, 8:520], y, tol)
    assert float((wide_o[:, :8] - MARK).abs().max()) == 0.0 and float((wide_o[:, 520:] - MARK).abs().max()) == 0.0


def test_bad_ranges_read_as_empty(gpu):
    """Ranges that the host cannot see: past the rows, negative, off a multiple of 8, longer than the limit."""
    import torch
    c = make(gpu, 11, "float16", 3, 1, 256, [9, 9, 9, 9], [24, 24, 24, 24], 30)
    c["k_start"] = torch.tensor([c["k"].shape[0] - 8, -8, c["ks"][2] + 4, c["ks"][3]], dtype=torch.int32, device=gpu)
    c["k_len"] = torch.tensor([24, 24, 16, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    c["k_lens"] = [0, 0, 0, 24]  # the last is cut to max_k
    got = _run(c, 0.0625)
    check(c, got, *reference(c, 0.0625, False))
    c["ctx"].fill_(MARK)
    c["q_start"] = torch.tensor([-1, c["Mq"] - 3, c["qs"][2], 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    c["liveq"][:] = False
    c["liveq"][c["qs"][2]:c["qs"][2] + 9] = True
    got = _run(c, 0.0625)
    y, tol = reference(c, 0.0625, False)
    check(c, got, y, tol)


def test_long_pitches_pass_32_bits(gpu):
    """V^T of a cache of 2^24 + 8 columns: a dim's offset passes 2^31 bytes within a head and 2^32 over the heads."""
    import torch
    cols = (1 << 24) + 8
    H, KV, D, n = 2, 2, 256, 40
    vt = torch.zeros((KV, D, cols), dtype=torch.float16, device=gpu)
    c = make(gpu, 12, "float16", H, KV, D, [n], [n], 20)
    k0 = cols - 48
    vt[:, :, k0:k0 + n] = c["vt"][:, :, c["ks"][0]:c["ks"][0] + n]
    y, tol = reference(c, 0.0625, False)
    big_k = torch.zeros((cols, KV * D), dtype=torch.float16, device=gpu)  # a row's offset passes 2^33 bytes
    big_k[k0:k0 + n] = c["k"][c["ks"][0]:c["ks"][0] + n]
    c["k"], c["vt"], c["k_start"] = big_k, vt, torch.tensor([k0], dtype=torch.int32, device=gpu)
    check(c, _run(c, 0.0625), y, tol)
    # single tokens take the same keys
    c["q_len"], c["q_lens"], c["max_q"] = torch.ones_like(c["q_len"]), [1], 1
    c["ctx"].fill_(MARK)
    c["liveq"][:] = False
    c["liveq"][c["qs"][0]] = True
    y[c["qs"][0] + 1:] = 0
    check(c, _run(c, 0.0625), y, tol)


def test_captured_replayed_and_two_streams(gpu):
    """A graph whose lengths change between replays, and two calls at once with a workspace each."""
    import e2mi
    import torch
    c = make(gpu, 13, "float16", 3, 1, 256, [1] * 6, [50] * 6, 500)
    _run(c, 0.0625)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run(c, 0.0625)
    for lens in ([50] * 6, [1, 2, 3, 4, 5, 6], [0, 50, 0, 50, 17, 33]):
        c["k_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        c["k_lens"] = lens
        c["ctx"].fill_(MARK)
        graph.replay()
        got = c["ctx"].clone()
        eager = _run(c, 0.0625, ctx=torch.full_like(c["ctx"], MARK))
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        check(c, got, *reference(c, 0.0625, False))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [torch.full_like(c["ctx"], MARK) for _ in range(2)]
    torch.cuda.synchronize()
    for s, o in zip((a, b), outs):
        for _ in range(4):
            e2mi.attention_prefix(c["q"], c["k"], c["vt"], c["pk"], c["pvt"], c["q_start"], c["q_len"], 1, 3, 1, k_start=c["k_start"],
                                  k_len=c["k_len"], max_k=c["max_k"], scale=0.0625, ctx=o, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)


def test_same_as_the_packed_attention_without_a_prefix(gpu):
    """Beside the framework's own attention: no prefix, its q16, k16, vt16 and ranges; both within the tolerance of the same
    64-bit context (the packed kernel's f32 copy)."""
    import e2mi
    c = make(gpu, 14, "float16", 3, 1, 256, [100, 40, 8], None, 0, lead=0)
    y, tol = reference(c, 0.0625, False)
    live = c["liveq"]
    q, k = c["q"].clone(), c["k"].clone()
    q[~live] = 0
    M = (q.shape[0] // 8) * 8
    vt = c["vt"][:, :, :M].clone()
    vt[:, :, ~live[:M]] = 0
    c32 = e2mi.attention_packed(q[:M], k[:M], vt.contiguous(), c["q_start"], c["q_len"], 100, 3, 1, scale=0.0625)[2]
    got = _run(c, 0.0625)
    check(c, got, y, tol)
    n = live[:M].cpu().numpy()
    assert np.all(np.abs(c32.double().cpu().numpy() - y[:M])[n] <= tol[:M][n])
