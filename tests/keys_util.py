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


def _f64(t):
    return t.double().cpu().numpy()


def reference(c, scale, causal, keys_of=None):
    """64-bit context and tolerance [Mq, H * D] (zeros outside the sequences). keys_of(b, token, kv head): the own
    keys a token reads, in any order (None: all)."""
    H, KV, D, G = c["H"], c["KV"], c["D"], c["H"] // c["KV"]
    q, k, vt = _f64(c["q"]), _f64(c["k"]), _f64(c["vt"])
    P = 0 if c["pk"] is None else c["pk"].shape[0]
    pk, pvt = (_f64(c["pk"]), _f64(c["pvt"])) if P else (np.zeros((0, KV * D)), np.zeros((KV, D, 0)))
    u = U[c["dtype"]]
    y, tol = np.zeros((c["Mq"], H * D)), np.zeros((c["Mq"], H * D))
    for b, (q0, k0, nq, nk) in enumerate(zip(c["qs"], c["ks"], c["q_lens"], c["k_lens"])):
        for a in range(KV):
            kk = np.concatenate([pk[:, a * D:(a + 1) * D], k[k0:k0 + nk, a * D:(a + 1) * D]])
            vv = np.concatenate([pvt[a].T, vt[a, :, k0:k0 + nk].T])
            for i in range(nq):
                own = np.arange(nk) if keys_of is None else np.asarray(keys_of(b, i, a), dtype=np.int64)
                own = own[own < nk]
                if causal:
                    own = own[own <= i + nk - nq]
                at = np.concatenate([np.arange(P), P + own])
                if not at.size:
                    continue
                rows = q[q0 + i].reshape(H, D)[a * G:(a + 1) * G]
                x = scale * rows @ kk[at].T
                L = (D + 4) * 2.0 ** -24 * scale * (np.abs(rows) @ np.abs(kk[at]).T).max(1, keepdims=True)
                p = np.exp(x - x.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                A = p @ np.abs(vv[at])
                o = p @ vv[at]
                t = A * (u + 2 * L + (at.size + 64) * 2.0 ** -24) + u * np.abs(o)
                if c["dtype"] == "float16":
                    t = t + at.size * 2.0 ** -25 * np.abs(vv[at]).max() + 2.0 ** -25
                y[q0 + i, a * G * D:(a + 1) * G * D] = o.ravel()
                tol[q0 + i, a * G * D:(a + 1) * G * D] = t.ravel()
    return y, tol


def check(c, got, want, tol):
    """Live rows within tolerance (a second rounding's worth of the tolerance on top), others untouched."""
    live = c["liveq"].cpu().numpy()
    g = _f64(got)
    assert np.all(g[~live] == MARK), "rows outside every sequence were written"
    off = np.abs(g - want)[live]
    t = (tol * (1 + U[c["dtype"]]))[live]
    assert off.size == 0 or np.all(off <= t), f"worst {np.max(off - t)} over the tolerance; largest off {np.nanmax(off)}"
