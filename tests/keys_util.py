"""Packed inputs and 64-bit references for the attention over a shared prefix and over selected blocks.

Rows outside every sequence hold NaN (q), keys outside hold NaN and infinities, output rows outside hold a
mark: nothing of them may reach a result, and the mark must stay.

Tolerance of a context value, from the arithmetic alone. With w = softmax weights and A = sum_j w_j |v_j|:
  probabilities rounded to the rows' type: half a step of each, A * u (u = 2^-11 f16, 2^-8 bf16), and for f16
  2^-25 absolute below its normal range, n keys of them against a sum of at least 1: n * 2^-25 * max |v|;
  logits: a dot of D products in f32 is off by at most (D + 4) * 2^-24 * scale * sum |q k|, its exponential by that
  relatively, once in the numerator and once in the sum: 2 * A * L; exp2, sums of n terms and the division stay under
  (n + 64) * 2^-24 * A;
  the output's own rounding: u * |y|."""
import numpy as np

U = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
MARK = 77.0


def starts(lens, step, lead=0):
    at, got = lead, []
    for n in lens:
        got.append(at)
        at += -(-max(n, 0) // step) * step
    return got, at


def make(dev, seed, dtype, H, KV, D, q_lens, k_lens, P=0, lead=8, spread=1.0):
    """A dict of device tensors; k_lens None: the same as q_lens (self-attention, one array of ranges)."""
    import torch
    g = torch.Generator(device=dev).manual_seed(seed)
    t = getattr(torch, dtype)
    same = k_lens is None
    k_lens = list(q_lens) if same else k_lens
    ks, Mk = starts(k_lens, 8, lead)
    qs, Mq = (ks, Mk) if same else starts(q_lens, 1, 3)
    Mk, Mq = Mk + 11, Mq + 5

    def randn(*s):
        return torch.randn(s, generator=g, device=dev)

    q, k = (spread * randn(Mq, H * D)).to(t), randn(Mk, KV * D).to(t)
    vt = randn(KV, D, Mk + 3).to(t)  # a pitch past the rows, odd for some sizes
    live = torch.zeros(Mk + 3, dtype=torch.bool, device=dev)
    liveq = torch.zeros(Mq, dtype=torch.bool, device=dev)
    for s, n in zip(ks, k_lens):
        live[s:s + n] = True
    for s, n in zip(qs, q_lens):
        liveq[s:s + n] = True
    k[~live[:Mk]] = float("nan")
    vt[:, :, ~live] = float("nan")
    vt[:, ::2, ~live] = float("inf")
    q[~liveq] = float("nan")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    c = dict(q=q, k=k, vt=vt, q_start=i32(qs), q_len=i32(q_lens), k_start=i32(ks), k_len=i32(k_lens), qs=qs, ks=ks,
             q_lens=list(q_lens), k_lens=list(k_lens), max_q=max(max(q_lens), 1), max_k=max(max(k_lens), 1), H=H, KV=KV, D=D,
             Mq=Mq, liveq=liveq, ctx=torch.full((Mq, H * D), MARK, dtype=t, device=dev), dtype=dtype)
    c["pk"] = randn(P, KV * D).to(t) if P else None
    c["pvt"] = randn(KV, D, P).to(t) if P else None
    return c


def reference(c, scale, causal, keys_of=None, q_block=None):
    """64-bit context and tolerance [Mq, H * D] (zeros outside the sequences), on the tensors' device. keys_of(b, block, kv head):
    the own keys (in any order, a key twice counts twice) that the block of q_block queries reads; None: all."""
    import torch
    H, KV, D, G = c["H"], c["KV"], c["D"], c["H"] // c["KV"]
    dev = c["q"].device
    f64 = dict(dtype=torch.float64, device=dev)
    u = U[c["dtype"]]
    y, tol = torch.zeros((c["Mq"], H * D), **f64), torch.zeros((c["Mq"], H * D), **f64)
    P = 0 if c["pk"] is None else c["pk"].shape[0]
    for b, (q0, k0, nq, nk) in enumerate(zip(c["qs"], c["ks"], c["q_lens"], c["k_lens"])):
        step = q_block or max(nq, 1)
        for a in range(KV):
            kk = [] if c["k"] is None else [c["k"][k0:k0 + nk, a * D:(a + 1) * D].double()]
            vv = [] if c["k"] is None else [c["vt"][a, :, k0:k0 + nk].double().T]
            if P:
                kk, vv = [c["pk"][:, a * D:(a + 1) * D].double()] + kk, [c["pvt"][a].double().T] + vv
            if not kk:
                continue
            kk, vv = torch.cat(kk).contiguous(), torch.cat(vv).contiguous()
            for i in range(0, nq, step):
                n = min(step, nq - i)
                own = torch.arange(nk, device=dev) if keys_of is None else torch.as_tensor(keys_of(b, i // step, a), dtype=torch.int64, device=dev)
                own = own[own < nk]
                at = torch.cat([torch.arange(P, device=dev), P + own])
                if not at.numel():
                    continue
                rows = c["q"][q0 + i:q0 + i + n].double().view(n, H, D)[:, a * G:(a + 1) * G].reshape(n * G, D)
                k, v = kk[at], vv[at]
                x = scale * (rows @ k.T.contiguous())
                last = (torch.arange(i, i + n, device=dev) + nk - nq if causal else torch.full((n,), nk, device=dev)).repeat_interleave(G)
                see = (at[None] < P) | (at[None] - P <= last[:, None])
                x = x.masked_fill(~see, -float("inf"))
                some = see.any(1, keepdim=True)
                L = (D + 4) * 2.0 ** -24 * scale * (rows.abs() @ k.abs().T.contiguous()).amax(1, keepdim=True)
                p = torch.exp(x - x.amax(1, keepdim=True).masked_fill(~some, 0.0))
                p = p / p.sum(1, keepdim=True).masked_fill(~some, 1.0)
                A, o = p @ v.abs(), p @ v
                t = A * (u + 2 * L + (at.numel() + 64) * 2.0 ** -24) + u * o.abs()
                if c["dtype"] == "float16":
                    t = t + (at.numel() * 2.0 ** -25 * v.abs().max() + 2.0 ** -25) * some
                y[q0 + i:q0 + i + n, a * G * D:(a + 1) * G * D] = o.reshape(n, G * D)
                tol[q0 + i:q0 + i + n, a * G * D:(a + 1) * G * D] = t.reshape(n, G * D)
    return y.cpu().numpy(), tol.cpu().numpy()


def _f64(t):
    return t.double().cpu().numpy()


def check(c, got, want, tol):
    """Live rows within tolerance (a second rounding's worth of the tolerance on top), others untouched."""
    live = c["liveq"].cpu().numpy()
    g = _f64(got)
    assert np.all(g[~live] == MARK), "rows outside every sequence were written"
    off = np.abs(g - want)[live]
    t = (tol * (1 + U[c["dtype"]]))[live]
    assert off.size == 0 or np.all(off <= t), f"worst {np.max(off - t)} over the tolerance; largest off {np.nanmax(off)}"


def route_prefix(c):
    """{apart, prefix: nw, shares, own keys: nw, shares, copies} that a call on c's sizes takes (attn_keys.hip)."""
    import ctypes as C
    import e2mi
    out = (C.c_int * 6)()
    e2mi.load()._ZN4e2mi17keys_route_prefixEiiiiiiiiiPi(c["Mq"], 0 if c["k"] is None else c["k"].shape[0],
                                                        0 if c["pk"] is None else c["pk"].shape[0], len(c["q_lens"]), c["max_q"],
                                                        c["max_k"], c["H"], c["KV"], c["D"], out)
    return list(out)


def route_blocks(c, q_block, n_sel):
    import ctypes as C
    import e2mi
    out = (C.c_int * 6)()
    e2mi.load()._ZN4e2mi17keys_route_blocksEiiiiiiiiiPi(c["Mq"], c["k"].shape[0], len(c["q_lens"]), c["max_q"], c["H"], c["KV"], c["D"], q_block,
                                                       n_sel, out)
    return list(out)
