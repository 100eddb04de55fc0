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
    return torch.logaddexp(x, torch.zeros((), dtype=x.dtype))


def attend(q, k, v, freqs, bias, lens, counts, scale, store=None):
    """q (b, h, n, d) in its type; k, v: lists of (hk, len, d) held values; -> out, lse, worst, rms (fp64, CPU)."""
    dt = q.dtype
    u_out = half_step(dt)
    b, h, n, d = q.shape
    hk, r = k[0].shape[0], freqs.shape[-1]
    # the type of the products' operands: that of q, but fp16 for an 8-bit cache and at most 16 rows of a key head
    u = half_step(torch.float16 if store is not None and n * h // hk <= 16 else dt)
    out = torch.zeros(b, h, n, d, dtype=torch.float64)
    lse = torch.full((b, h, n), -math.inf, dtype=torch.float64)
    worst, rms2 = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(b):
        ln, m = lens[i], counts[i]
        for row in range(m):
            pos = ln - m + row
            if pos < 0:
                continue
            for head in range(h):
                e = head % hk
                kk, vv, qq = k[i][e, :pos + 1].double().cpu(), v[i][e, :pos + 1].double().cpu(), q[i, head, row].double().cpu()
                f = freqs[:pos + 1].double().cpu()
                aq, ak = softplus(qq[:r]), softplus(kk[:, :r])
                rest = kk[:, r:] * qq[r:]
                s = scale * ((ak * aq * torch.cos(f[pos] - f - bias[e].double().cpu())).sum(-1) + rest.sum(-1))
                p = torch.softmax(s, 0)
                o = p @ vv
                both = torch.cat((aq * ak, aq * ak, rest.abs()), -1)
                ds = abs(scale) * both.sum(-1) * (4 * u + 2 ** -10)
                ds2 = scale ** 2 * both.square().sum(-1) * (4 * u * u + 2 * 2.0 ** -22) / 3
                out[i, head, row], lse[i, head, row] = o, torch.logsumexp(s, 0)
                worst[i, head, row] = 1.1 * (u_out * o.abs() + 2 * u * (p @ vv.abs()) + (p * ds) @ (vv.abs() + o.abs()))
                if ds2.max() > 1 / 64:
                    # scores that are off by an eighth and more: exp(ds) - 1 is no longer ds, and the first order says nothing (where one key
                    # has all of the weight it gives ds |v| of that key alone, while another key may take its place).  What holds: out is a
                    # mean of the rows of v whatever the scores are, so two of them differ by 2 max |v| at most, next to the other roundings.
                    far = 2 * vv.abs().max(0).values
                    worst[i, head, row], rms2[i, head, row] = 1.1 * (1 + u_out + 2 * u) * far, far ** 2
                    continue
                rms2[i, head, row] = (u_out * o) ** 2 / 3 + (p * p) @ vv.square() * 2 * u * u / 3 + (p * p * ds2) @ (vv - o).square()
    return out, lse, worst, rms2.sqrt()


def check(got, want, worst, rms, lse=None, want_lse=None):
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    # (2^-24: results next to zero, where the type's smallest steps are what is left)
    assert (err <= worst + 2.0 ** -24).all(), (err - worst).max().item()
    assert err.norm() <= 2 * rms.norm() + 1e-6, (err.norm().item(), rms.norm().item())
    if lse is not None:
        lse = lse.double().cpu()
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isneginf(lse), empty)
        # the scores' errors, at most: bounded through out's own bound by the largest of them
        assert (lse - want_lse)[~empty].abs().max().item() <= 0.1 if (~empty).any() else True
