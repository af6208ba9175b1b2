"""The bf16 backward of packed attention with each of its roundings and everything else in 64 bits: what the error of dQ
and dK over their norm is, with dS in two bf16 parts or one, and with delta from f32 sums or from the rounded output."""
import torch

F64 = torch.float64


def bf16(x):
    """Rounded once to bf16 (through f32: what the kernels hold)."""
    return x.float().to(torch.bfloat16).to(F64)


def two_parts(x):
    x = x.float()
    hi = (x.view(torch.int32) & -65536).view(torch.float32)
    return hi.to(F64) + (x - hi).to(torch.bfloat16).to(F64)


def case(lens, hq, hkv, D, seed, keys=0.0, values=0.0, device="cpu"):
    """A batch whose keys, or values, share a direction, as trained ones do. dS sums to zero along a row: with the keys'
    direction dQ is a small difference of large terms, and with the values' delta is large beside the differences."""
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    q, do = torch.randn(n, hq, D, generator=g) * 1.2, torch.randn(n, hq, D, generator=g) * 0.1
    k, v = torch.randn(n, hkv, D, generator=g), torch.randn(n, hkv, D, generator=g)
    k, v = k + keys * torch.randn(1, hkv, D, generator=g), v + values * torch.randn(1, hkv, D, generator=g)
    return [x.to(torch.bfloat16).to(device) for x in (q, k, v, do)]


def gradients(q, k, v, do, lens, causal):
    """{name: (exact, as the kernels round, with the coarser rounding)} of dq and dk."""
    n, hq, D = q.shape
    hkv, scale = k.shape[1], D ** -0.5
    G = hq // hkv
    r = {x: [torch.zeros(n, h, D, dtype=F64, device=q.device) for _ in range(3)] for x, h in (("dq", hq), ("dk", hkv))}
    lo = 0
    for m in lens:
        s = slice(lo, lo + m)
        lo += m
        for h in range(hq):
            Q, K, V, dO = (x.to(F64) for x in (q[s, h], k[s, h // G], v[s, h // G], do[s, h]))
            a = Q @ K.T * scale
            if causal:
                a = a.masked_fill(torch.ones(m, m, dtype=torch.bool, device=q.device).triu(1), -torch.inf)
            P = torch.softmax(a, 1)
            dP = dO @ V.T
            delta = (P * dP).sum(1, keepdim=True)
            rounded = (dO * bf16(bf16(P) @ V)).sum(1, keepdim=True)     # from the stored output
            dS, dSr = P * (dP - delta), P * (dP - rounded)
            for i, x in enumerate((dS, two_parts(dSr), bf16(dSr))):
                r["dq"][i][s, h] = x @ K * scale
            for i, x in enumerate((dS, bf16(dS), bf16(dSr))):
                r["dk"][i][s, h // G] += x.T @ Q * scale
    return {name: (x[0], bf16(x[1]), bf16(x[2])) for name, x in r.items()}


def error(x, exact):
    return float((x.to(F64) - exact).norm() / exact.norm())
