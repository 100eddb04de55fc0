"""What the paged cache's operators compute, in 64 bits, and how far 16-bit operands may be from it.

The bounds follow from the roundings.  u = half a step of a type relative to the value (bf16 2^-8, fp16 2^-11).  Each expanded
operand q', k' is rounded at most twice (the magnitude and its product with a cosine or sine) and its cosine or sine carries one
more rounding, of an fp16 table (2^-11); so a product q'_c k'_c is off by at most (4 u + 2 * 2^-11) of the product of the
magnitudes.  To first order an error ds_j of the scores moves out by sum_j p_j ds_j (v_j - out); the probabilities are rounded
once before they meet v (u), v itself once more where it is held in 8 bits, and out is rounded once to its type.
``worst`` adds all of these up as they could at most come together, with a tenth for the second order.  ``rms`` takes them as independent
and evenly spread over their intervals (1 / sqrt(3) of the bound each): what the 2-norm of a right result's error comes to."""
import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def softplus(x):
    return torch.logaddexp(x, torch.zeros((), dtype=x.dtype, device=x.device))


def attend(q, k, v, freqs, bias, lens, counts, scale, store=None):
    """q (b, h, n, d) in its type; k, v: lists of (hk, len, d) held values; -> out, lse, worst, rms (fp64, on q's device)."""
    dt, dev = q.dtype, q.device
    u_out = half_step(dt)
    b, h, n, d = q.shape
    hk, r = k[0].shape[0], freqs.shape[-1]
    # the type of the products' operands: that of q, but fp16 for an 8-bit cache and at most 16 rows of a key head
    u = half_step(torch.float16 if store is not None and n * h // hk <= 16 else dt)
    out = torch.zeros(b, h, n, d, dtype=torch.float64, device=dev)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64, device=dev)
    worst, rms2 = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(b):
        ln, m = lens[i], counts[i]
        skip = max(0, m - ln)          # rows at negative positions
        if m - skip <= 0:
            continue
        pos = torch.arange(ln - m + skip, ln, device=dev)
        for e in range(hk):
            kk, vv, qq = k[i][e, :ln].double(), v[i][e, :ln].double(), q[i, e::hk, skip:m].double()     # qq: (group, rows, d)
            f, beta = freqs[:ln].double(), bias[e].double()
            aq, ak = softplus(qq[..., :r]), softplus(kk[:, :r])
            qc, qs = aq * torch.cos(freqs[pos].double()), aq * torch.sin(freqs[pos].double())
            s = qc @ (ak * torch.cos(f + beta)).T + qs @ (ak * torch.sin(f + beta)).T + qq[..., r:] @ kk[:, r:].T
            s = (scale * s).masked_fill(torch.arange(ln, device=dev) > pos[:, None], -math.inf)
            p = torch.softmax(s, -1)
            o = p @ vv
            both = 2 * aq @ ak.T + qq[..., r:].abs() @ kk[:, r:].abs().T
            both2 = 2 * aq.square() @ ak.square().T + qq[..., r:].square() @ kk[:, r:].square().T
            ds = abs(scale) * both * (4 * u + 2 ** -10)
            ds2 = scale ** 2 * both2 * (4 * u * u + 2 * 2.0 ** -22) / 3
            near = u_out * o.abs() + 2 * u * (p @ vv.abs())
            w = 1.1 * (near + (p * ds) @ vv.abs() + (p * ds).sum(-1, keepdim=True) * o.abs())
            pd = p * p * ds2
            r2 = (u_out * o) ** 2 / 3 + (p * p) @ vv.square() * 2 * u * u / 3 + pd @ vv.square() - 2 * (pd @ vv) * o + pd.sum(-1, keepdim=True) * o.square()
            # Scores that are off by an eighth and more: exp(ds) - 1 is no longer ds, and the first order says nothing (where one key has all of the
            # weight it gives ds |v| of that key alone, while another key may take its place).  What holds: out is a mean of the rows of v
            # whatever the scores are, so two of them differ by 2 max |v| at most, next to the other roundings.
            wild = (ds2.masked_fill(torch.isinf(s), 0).amax(-1, keepdim=True) > 1 / 64)
            far = (2 * vv.abs().amax(0)).expand_as(o)
            at = (i, slice(e, None, hk), slice(skip, m))
            out[at], lse[at] = o, torch.logsumexp(s, -1)
            worst[at], rms2[at] = torch.where(wild, 1.1 * (1 + u_out + 2 * u) * far, w), torch.where(wild, far ** 2, r2.clamp(min=0))
    return out, lse, worst, rms2.sqrt()


def check(got, want, worst, rms, lse=None, want_lse=None):
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    # (2^-24: results next to zero, where the type's smallest steps are what is left)
    assert (err <= worst + 2.0 ** -24).all(), (err - worst).max().item()
    assert err.norm() <= 2 * rms.norm() + 1e-6, (err.norm().item(), rms.norm().item())
    if lse is not None:
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isneginf(lse), empty)
        # the scores' errors, at most: bounded through out's own bound by the largest of them
        assert (lse - want_lse)[~empty].abs().max().item() <= 0.1 if (~empty).any() else True
