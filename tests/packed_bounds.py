"""64-bit reference of attention over packed sequences under masks of any size, with the error that its kernels may have:
as packed_reference.py, element by element from the formulas, but closer.

A score is off by what its own terms and the row's lse round off; what a key far below the row's maximum (by more than
200, a probability of e^-200) rounds off does not count, so a large finite mask does not widen the bound of the rows
that see other keys: e_s = (D + 8) 2^-24 (max over the near keys of (scale |q|.|k| + |g b|) + |lse| + 72), 72 for the
distance between a score and the reference that the kernels take it relative to (2^6 + 2^3). dS goes into dQ in two bf16
parts (the rest after its upper 16 bits, less than 2^-7 of it, is off by 2^-8 of itself: 2^-15), and dK takes delta from
f32 sums for every bf16 call. A row under a bias whose largest score is below -2^14 is left nothing."""
import torch

from packed_reference import F64, TINY, U, sequences

LEAST = -16384.0


def reference(q, k, v, cu, *, causal, scale=None, used=None, gate=None, vec=None, dout=None):
    """-> {name: (value, bound)}; rows of no sequence, and rows whose largest score lies within 1 % of -2^14, hold NaN
    (in dk, dv and dvec such rows are counted in: a caller has none)."""
    rows, hq, D = q.shape
    hkv, dev = k.shape[1], q.device
    G = hq // hkv
    b16 = q.dtype == torch.bfloat16
    h = 2.0 ** -8 if b16 else 2.0 ** -24
    hq2 = 2.0 ** -15 if b16 else 2.0 ** -24
    scale = D ** -0.5 if scale is None else scale
    nul = torch.zeros((), dtype=F64, device=dev)

    def new(*shape, fill=float("nan")):
        return torch.full(shape, fill, dtype=F64, device=dev), torch.full(shape, fill, dtype=F64, device=dev)

    r = {"out": new(rows, hq, D), "lse": new(hq, rows)}
    T = 0 if vec is None else (vec.shape[1] + 1) // 2
    if dout is not None:
        r.update(dq=new(rows, hq, D), dk=new(rows, hkv, D), dv=new(rows, hkv, D))
        if vec is not None:
            r["dvec"] = new(hq, 2 * T - 1, fill=0.0)
            if gate is not None:
                r["dgate"] = new(hq, rows)
    for lo, hi in sequences(cu, used):
        n = hi - lo
        if n == 0:
            continue
        i, j = torch.arange(n, device=dev)[:, None], torch.arange(n, device=dev)[None, :]
        at = (j - i + T - 1).clamp(0, max(2 * T - 2, 0))
        gam = (n + D + 16) * U
        for hh in range(hq):
            c = hh // G
            Q, K, V = q[lo:hi, hh].to(F64), k[lo:hi, c].to(F64), v[lo:hi, c].to(F64)
            s, mag = Q @ K.T * scale, Q.abs() @ K.abs().T * abs(scale)
            if vec is not None:
                b = vec[hh].to(F64)[at]
                g = torch.ones(n, 1, dtype=F64, device=dev) if gate is None else gate[hh, lo:hi].to(F64)[:, None]
                s, mag = s + g * b, mag + (g * b).abs()
            if causal:
                s = torch.where(j <= i, s, -float("inf"))
            top = s.amax(1, keepdim=True)
            empty = torch.isinf(top)
            if vec is not None:
                empty = empty | (top < LEAST)
                unsure = ((top / LEAST - 1).abs() < 0.01)[:, 0]
            else:
                unsure = torch.zeros(n, dtype=torch.bool, device=dev)
            lse = torch.where(empty, nul, torch.logsumexp(s, 1, keepdim=True))
            P = torch.where(empty, nul, torch.exp(s - lse))
            near = (s > lse - 200) & ~empty
            es = (D + 8) * U * (torch.where(near, mag, nul).amax(1, keepdim=True) + lse.abs() + 72)
            ep = 2 * es + 2.0 ** -21
            O = P @ V
            eO = (ep + h + gam) * (P @ V.abs()) * 1.01 + h * O.abs() + TINY * V.abs().sum(0, keepdim=True)
            r["out"][0][lo:hi, hh], r["out"][1][lo:hi, hh] = O, eO
            r["lse"][0][hh, lo:hi] = torch.where(empty, -torch.inf, lse)[:, 0]
            r["lse"][1][hh, lo:hi] = torch.where(empty, nul, ep + gam)[:, 0]
            r["out"][0][lo:hi, hh][unsure] = float("nan")
            r["lse"][0][hh, lo:hi][unsure] = float("nan")
            if dout is None:
                continue
            dO = dout[lo:hi, hh].to(F64)
            dP, mdP = dO @ V.T, dO.abs() @ V.abs().T
            delta = (P * dP).sum(1, keepdim=True)
            mdl = (P * mdP).sum(1, keepdim=True)
            dS = P * (dP - delta)
            flush = TINY * (1 + mdP + delta.abs())
            e_sum = (ep + 2 * gam) * mdl
            e_out = (dO.abs() * eO).sum(1, keepdim=True) + gam * mdl
            eds = (ep + 2 * U) * P * (dP - delta).abs() + gam * P * mdP + flush

            def e_dS(ed, hs):
                return (eds + P * ed) * (1 + hs) + hs * dS.abs()

            dV = P.T @ dO
            e_q, e_k = e_dS(e_out, hq2), e_dS(e_sum if b16 or vec is not None else e_out, h)
            dQ, dK = dS @ K * scale, dS.T @ Q * scale
            r["dq"][0][lo:hi, hh] = dQ
            r["dq"][1][lo:hi, hh] = abs(scale) * ((e_q + gam * dS.abs()) @ K.abs()) * 1.01 + h * dQ.abs() + 2 * U * dQ.abs()
            r["dq"][0][lo:hi, hh][unsure] = float("nan")
            eK = abs(scale) * ((e_k + G * gam * dS.abs()).T @ Q.abs()) * 1.01
            eV = ((ep + h + G * gam) * P + TINY).T @ dO.abs() * 1.01
            for name, val, err in (("dk", dK, eK), ("dv", dV, eV)):
                if hh % G == 0:
                    r[name][0][lo:hi, c], r[name][1][lo:hi, c] = 0.0, 0.0
                r[name][0][lo:hi, c] += val
                r[name][1][lo:hi, c] += err
                if hh % G == G - 1:
                    r[name][1][lo:hi, c] += h * r[name][0][lo:hi, c].abs()
            if vec is not None:
                bp = torch.where(P > 0, b, nul)      # (a key without a probability adds nothing, whatever its bias)
                if gate is not None:
                    r["dgate"][0][hh, lo:hi] = (dS * bp).sum(1)
                    m1 = (P * mdP * bp.abs()).sum(1) + mdl[:, 0] * (P * bp.abs()).sum(1)
                    r["dgate"][1][hh, lo:hi] = (2 * ep[:, 0] + 4 * gam) * m1 + (flush * bp.abs()).sum(1)
                    r["dgate"][0][hh, lo:hi][unsure] = float("nan")
                gd = g * dS
                egd = g.abs() * (eds + P * e_sum) * 1.01
                idx = (j - i + T - 1).reshape(-1)
                r["dvec"][0][hh].index_add_(0, idx, gd.reshape(-1))
                r["dvec"][1][hh].index_add_(0, idx, (egd + (rows + 64) * U * gd.abs()).reshape(-1))
    return r
