"""Plain restatement of attention within a window on the CPU, in 64 bits (test infrastructure only), from the
definition in include/dsqg.h, with bounds for a kernel's roundings."""

import torch


def sees(N, window, sinks, length=None):
    """[N, N] bool: row i sees column j."""
    i, j = torch.arange(N)[:, None], torch.arange(N)[None]
    n = N if length is None else max(0, min(N, length))
    return (j <= i) & ((i - j < window) | (j < sinks)) & (i < n)


def attend(q, k, v, window, sinks=0, length=None, scale=None):
    """out [N, D] of one head, differentiable."""
    s = (q @ k.T) * (q.shape[1] ** -0.5 if scale is None else scale)
    m = sees(q.shape[0], window, sinks, length)
    p = torch.softmax(s.masked_fill(~m, -torch.inf), dim=-1)
    return torch.where(m.any(-1, keepdim=True), p, 0.0) @ v


def forward_backward(q, k, v, dout, window, sinks=0, lengths=None, scale=None):
    """({out, dq, dk, dv}, bounds of the same shapes) of q, dout [B,H,N,D], k, v [B,Hkv,N,D].

    The bounds, u = 2^-24, e half a step of the 16-bit type (0 for float32), t the result's half step:
    * a score's D products, its scaling, the difference to the maximum, whose magnitude is at most twice the largest
      score's `size` = |scale| sum |q||k|, and 2^x: a weight is (D + 7) u size + 2 u off, the normalised one twice that
      (in the backward, whose scores may come from another order of sums, twice that again): r;
    * out: r, e of each weight (float16: 2^-38 of the largest where the weight is subnormal: weights are taken times
      2^14), 2 N u for its sums, relative to P |v|;
    * D_i = dout . out, of the stored out: |dout| times out's bound, (D + 2) u |dout||out|;
    * dS: (e + r) |dS| + p ((D + 2) u |dout||v| + the bound of D_i); float16's smallest step, 2^-25;
    * dq, dk, dv: sums of those bounds times the other factor, 2 N G u for the sums.
    Last, each result's rounding.
    """
    dt = q.dtype
    u, fi = 2.0 ** -24, torch.finfo(dt)
    e = 0.0 if dt == torch.float32 else fi.eps / 2
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    B, H, N, D = q.shape
    Hkv = k.shape[1]
    G = H // Hkv
    c = D ** -0.5 if scale is None else scale
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    ref = {n: torch.zeros_like(x) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(x) for n, x in ref.items()}

    def rounded(x, t):
        return t + (x.abs() + t) * (fi.eps / 2) + fi.smallest_normal * fi.eps

    for b in range(B):
        m = sees(N, window, sinks, None if lengths is None else int(lengths[b]))
        for h in range(H):
            x, kk, vv, do = q[b, h], k[b, h // G], v[b, h // G], dout[b, h]
            live = m.any(-1, keepdim=True)
            s = (x @ kk.T * c).masked_fill(~m, -torch.inf)
            p = torch.where(live, torch.softmax(s, dim=-1), 0.0)
            size = (x.abs() @ kk.abs().T * abs(c)).masked_fill(~m, 0.0).amax(-1, keepdim=True)
            out = p @ vv
            r = 2 * ((D + 7) * u * size + 2 * u)
            top = p.amax(-1, keepdim=True)
            t_out = (p @ vv.abs()) * (r + e * (1 + 2 * e) + 2 * (N + 8) * u)
            if tiny:
                t_out = t_out + top * (m.double() @ vv.abs()) * 2.0 ** -38
            ref["out"][b, h], tol["out"][b, h] = out, torch.where(live, rounded(out, t_out), 0.0)
            do = torch.where(live, do, 0.0)
            dp = do @ vv.T
            delta = (do * out).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            t_delta = (do.abs() * (tol["out"][b, h] + (D + 2) * u * out.abs())).sum(-1, keepdim=True)
            t_p = p * (2 * r + e) + m * tiny
            t_ds = ds.abs() * (2 * r + e) + p * ((D + 2) * u * (do.abs() @ vv.abs().T) + t_delta) * (1 + e) + m * tiny
            n = 2 * (N * G + 8) * u
            ref["dq"][b, h] = ds @ kk * c
            tol["dq"][b, h] = rounded(ref["dq"][b, h], ((t_ds + ds.abs() * n) @ kk.abs()) * abs(c))
            ref["dk"][b, h // G] += ds.T @ x * c
            tol["dk"][b, h // G] += ((t_ds + ds.abs() * n).T @ x.abs()) * abs(c)
            ref["dv"][b, h // G] += p.T @ do
            tol["dv"][b, h // G] += (t_p + p * n).T @ do.abs()
    for name in ("dk", "dv"):
        tol[name] = rounded(ref[name], tol[name])
    return ref, tol
