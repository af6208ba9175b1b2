"""64-bit reference of attention over packed sequences, with the error that its kernels may have.

Bounds, element by element, from the formulas: a rounding to bf16 is off by at most h = 2^-8 of the value (none in
f32), a sum of n f32 terms by at most n 2^-24 of the sum of their magnitudes, and a score by
e_s = (D + 8) 2^-24 (scale |q|.|k| + |g b| + |lse|), which is the relative error of its probability (twice: the
score's and the row's lse), beside 2^-21 of the exponential and the division. A probability below f32's least
normal number may be flushed: it is off by at most 2^-126, and what it multiplies carries that on."""
import torch

F64 = torch.float64
U = 2.0 ** -24
TINY = 2.0 ** -126


def sequences(cu, used):
    cu = cu.tolist()
    return [(a, (b if used is None else a + int(used[i]))) for i, (a, b) in enumerate(zip(cu[:-1], cu[1:]))]


def reference(q, k, v, cu, *, causal, scale=None, used=None, gate=None, vec=None, dout=None):
    """-> {name: (value, bound)}: out, lse and, with dout, dq, dk, dv, dgate, dvec; rows of no sequence hold NaN."""
    rows, hq, D = q.shape
    hkv, dev = k.shape[1], q.device
    G = hq // hkv
    h = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -24
    scale = D ** -0.5 if scale is None else scale

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
        gam = (n + D + 16) * U          # the sums over keys, rows and dims
        for hh in range(hq):
            c = hh // G
            Q, K, V = q[lo:hi, hh].to(F64), k[lo:hi, c].to(F64), v[lo:hi, c].to(F64)
            s, mag = Q @ K.T * scale, Q.abs() @ K.abs().T * abs(scale)
            if vec is not None:
                b = vec[hh].to(F64)[at]
                g = torch.ones(n, 1, dtype=F64, device=dev) if gate is None else gate[hh, lo:hi].to(F64)[:, None]
                s, mag = s + g * b, mag + (g * b.clamp(min=-1e30)).abs().where(b > -1e30, torch.zeros((), dtype=F64, device=dev))
            if causal:
                s = torch.where(j <= i, s, -float("inf"))
            lse = torch.logsumexp(s, 1, keepdim=True)
            empty = torch.isinf(lse)
            P = torch.where(empty, torch.zeros((), dtype=F64, device=dev), torch.exp(s - torch.where(empty, torch.zeros_like(lse), lse)))
            live = s > -float("inf")
            es = (D + 8) * U * (torch.where(live, mag, torch.zeros_like(mag)).amax(1, keepdim=True)
                                + torch.where(empty, torch.zeros_like(lse), lse.abs()))
            ep = 2 * es + 2.0 ** -21
            O = P @ V
            eO = (ep + h + gam) * (P @ V.abs()) * 1.01 + h * O.abs() + TINY * V.abs().sum(0, keepdim=True)
            r["out"][0][lo:hi, hh], r["out"][1][lo:hi, hh] = O, eO
            r["lse"][0][hh, lo:hi] = lse[:, 0]
            r["lse"][1][hh, lo:hi] = torch.where(empty, torch.zeros_like(lse), ep + gam)[:, 0]
            if dout is None:
                continue
            dO = dout[lo:hi, hh].to(F64)
            dP, mdP = dO @ V.T, dO.abs() @ V.abs().T
            delta = (P * dP).sum(1, keepdim=True)
            mdl = (P * mdP).sum(1, keepdim=True)
            dS = P * (dP - delta)
            # delta from the stored (rounded) output, or, beside a bias, from f32 sums
            e_sum = (ep + 2 * gam) * mdl
            e_out = (dO.abs() * eO).sum(1, keepdim=True) + gam * mdl
            eds = (ep + 2 * U) * P * (dP - delta).abs() + gam * P * mdP + TINY * (1 + mdP + delta.abs())

            def e_dS(ed):
                return (eds + P * ed) * (1 + h) + h * dS.abs()

            dV = P.T @ dO
            e_q, e_k = e_dS(e_out), e_dS(e_out if vec is None else e_sum)
            dQ, dK = dS @ K * scale, dS.T @ Q * scale
            r["dq"][0][lo:hi, hh] = dQ
            r["dq"][1][lo:hi, hh] = abs(scale) * ((e_q + gam * dS.abs()) @ K.abs()) * 1.01 + h * dQ.abs() + 2 * U * dQ.abs()
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
                bf = torch.where(b > -1e30, b, torch.zeros_like(b))
                if gate is not None:
                    r["dgate"][0][hh, lo:hi] = (dS * bf).sum(1)
                    m1 = (P * mdP * bf.abs()).sum(1) + mdl[:, 0] * (P * bf.abs()).sum(1)
                    r["dgate"][1][hh, lo:hi] = (2 * ep[:, 0] + 4 * gam) * m1
                gd = g * dS
                egd = g.abs() * (eds + P * e_sum) * 1.01
                idx = (j - i + T - 1).reshape(-1)
                r["dvec"][0][hh].index_add_(0, idx, gd.reshape(-1))
                r["dvec"][1][hh].index_add_(0, idx, (egd + (rows + 64) * U * gd.abs()).reshape(-1))
    return r


def worst(got, ref):
    """The largest error over its bound (rows of no sequence left out); 2^-126 is where f32 ends."""
    val, err = ref
    m = ~torch.isnan(val)
    g, val, err = got.to(F64)[m], val[m], err[m]
    if g.numel() == 0:
        return 0.0
    same = g == val        # infinities
    d = torch.where(same, torch.zeros_like(val), (g - val).abs())
    return float((d / (err + TINY)).max())
