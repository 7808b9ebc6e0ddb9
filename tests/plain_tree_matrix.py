"""The gated delta rule over one tree in matrix form, in 64 bits, with first-order bounds of its 32-bit evaluation by block doubling.

With A strictly lower (``A_ji = -beta_j e^{c_j - c_i} k_j.k_i`` above j), the updates are ``D = (1 - A)^-1 W`` and the outputs ``e^c q^T S0 + B D``.
The products ``1 - beta k k^T`` along a path never lengthen a vector, so entries of the inverse and of what it is built from are at most 1
however equal the keys are; a bound that follows the errors of the substitution node by node doubles with every node instead, and says nothing
after a run of one token.  Here the errors of each block product are added as they are made.
"""
import torch

from plain_tree import RING, U32, UBF, path_of


def gdn(proj, conv_w, A_log, dt_bias, norm_w, ring, state, pos0, parents, nk, nv, dk, dv, eps):
    """(out, bound, updates, bound), each ``[C, nv, dv]``: ``proj [C, width]``, ``ring [16, conv]`` and ``state [nv, dk, dv]`` of the sequence."""
    C, dev = len(parents), proj.device
    conv, rep = 2 * nk * dk + nv * dv, nv // nk
    n_eps = (2 * dk + C + 64) * U32
    x = torch.zeros(C, conv, dtype=torch.float64, device=dev)
    xe = torch.zeros_like(x)
    on = torch.zeros(C, C, dtype=torch.float64, device=dev)
    for j in range(C):
        path = path_of(parents, j)
        on[j, path] = 1
        lines = [ring[p % RING].double() for p in range(max(0, pos0 - 3), pos0)] + [proj[i, :conv].double() for i in path]
        lines = [torch.zeros(conv, dtype=torch.float64, device=dev)] * max(0, 4 - len(lines)) + lines[-4:]
        x[j] = sum(lines[t] * conv_w[:, t].double() for t in range(4))
        xe[j] = 1.1 * sum(lines[t].abs() * conv_w[:, t].double().abs() for t in range(4)) * 8 * U32
    x = x * torch.sigmoid(x)

    def unit(lo, scale):
        t, e = (y[:, lo:lo + nk * dk].reshape(C, nk, dk) for y in (x, xe))
        n = torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6)
        err = e / n + t.abs() / n * ((t.abs() * e).sum(-1, keepdim=True) / n ** 2 + (dk + 8) * U32)
        return [(y * scale).repeat_interleave(rep, 1).transpose(0, 1) for y in (t / n, err)]      # [nv, C, dk]

    (q, qe), (k, ke) = unit(0, dk ** -0.5), unit(nk * dk, 1.0)
    v, ve = (y[:, 2 * nk * dk:].reshape(C, nv, dv).transpose(0, 1) for y in (x, xe))
    rest = proj[:, conv:].double()
    z = rest[:, :nv * dv].reshape(C, nv, dv).transpose(0, 1)
    beta = torch.sigmoid(rest[:, nv * dv:nv * dv + nv]).T                                             # [nv, C]
    g = (-torch.exp(A_log.double()) * torch.nn.functional.softplus(rest[:, nv * dv + nv:nv * dv + 2 * nv] + dt_bias.double(), threshold=1e9)).T
    c = g @ on.T
    dec = torch.exp(c)
    S = state.double()

    def from_state(y, e):
        val, mag = dec[..., None] * (y @ S), dec[..., None] * (y.abs() @ S.abs())
        return val, mag * (n_eps + 8 * U32 * c.abs())[..., None] + dec[..., None] * (e @ S.abs())

    def gram(y, e, mask):
        diff = c[:, :, None] - c[:, None, :]
        f = torch.exp(torch.where(mask > 0, diff, torch.zeros_like(diff))) * mask
        mag = y.abs() @ k.abs().transpose(1, 2)
        return f * (y @ k.transpose(1, 2)), f * (mag * (n_eps + 8 * U32 * diff.abs()) + e @ k.abs().transpose(1, 2) + y.abs() @ ke.transpose(1, 2))

    A, Ae = gram(k, ke, on - torch.eye(C, dtype=torch.float64, device=dev))
    A, Ae = -beta[..., None] * A, beta[..., None] * Ae + 8 * U32 * (beta[..., None] * A).abs()
    B, Be = gram(q, qe, on)
    w, we = from_state(k, ke)
    W = beta[..., None] * (v - w)
    We = beta[..., None] * (ve + we) + (beta[..., None] * (v.abs() + w.abs())) * n_eps
    P = (C + 7) // 8 * 8
    eye = torch.eye(P, dtype=torch.float64, device=dev)
    Ap = torch.nn.functional.pad(A, (0, P - C, 0, P - C))
    M = torch.linalg.solve_triangular(eye - Ap, eye.expand(nv, P, P), upper=False, unitriangular=True)
    E = torch.zeros_like(M)
    for p in range(0, P, 4):                          # a column by substitution: at most as off as with all terms of one sign
        s = slice(p, p + 4)
        E[:, s, s] = 8 * U32 * (torch.linalg.solve_triangular(torch.eye(4, dtype=torch.float64, device=dev) - Ap[:, s, s].abs(),
                                                              torch.eye(4, dtype=torch.float64, device=dev).expand(nv, 4, 4), upper=False, unitriangular=True)
                             - torch.eye(4, dtype=torch.float64, device=dev))
    n = 4
    while n < P:                                      # M21 = M22 (A21 M11)
        for p in range(0, P - n, 2 * n):
            lo, hi = slice(p, p + n), slice(p + n, min(P, p + 2 * n))
            T = Ap[:, hi, lo] @ M[:, lo, lo]
            Te = Ap[:, hi, lo].abs() @ ((n + 4) * U32 * M[:, lo, lo].abs() + E[:, lo, lo])
            E[:, hi, lo] = M[:, hi, hi].abs() @ (Te + (n + 4) * U32 * T.abs()) + E[:, hi, hi] @ T.abs()
        n *= 2
    M, E = M[:, :C, :C], E[:, :C, :C]
    E = E + M.abs() @ Ae @ M.abs()
    D = M @ W
    De = E @ W.abs() + M.abs() @ (We + (C + 8) * U32 * W.abs())
    o, oe = from_state(q, qe)
    oe = oe + Be @ D.abs() + B.abs() @ (De + (C + 8) * U32 * D.abs()) + o.abs() * n_eps
    o = o + B @ D
    rms = torch.sqrt((o * o).mean(-1, keepdim=True) + eps)
    f = norm_w.double() * z * torch.sigmoid(z) / rms
    out = o * f
    oute = oe * f.abs() + out.abs() * ((o.abs() * oe).mean(-1, keepdim=True) / rms ** 2 + (dv + 64) * U32) + out.abs() * UBF
    return tuple(y.transpose(0, 1) for y in (out, oute * 1.01 + 1e-30, D, De * 1.01 + 1e-30))
