"""Gradients of a bias against the sum, in 64 bits, of the very terms that the kernels add up."""

import torch


def depth(rows, in_part, splits):
    """Additions that one term passes through: `in_part` in the CTA that leaves a part, then the parts' rows in turn to 32 warps of
    `splits` CTAs, a sum over lanes and one over the CTAs."""
    return in_part + -(-rows // (32 * splits)) + 5 + splits


def check(got, terms, additions, rows=None):
    """got [...] = the sum of terms [n, ...] over n; each addition rounds by 2^-24 of a partial sum, which the sizes bound. `rows`: the
    length of the parts; losing one of them has to show, or the comparison says nothing."""
    t = got.detach().cpu()
    terms = terms.detach().cpu().double()
    want, limit = terms.sum(0), additions * 2.0 ** -24 * terms.abs().sum(0)
    off = (t.double() - want).abs() - limit - torch.finfo(t.dtype).eps / 2 * (want.abs() + limit)
    assert off.max() <= 0, (off.max().item(), limit.max().item())
    if rows is not None:
        lost = torch.stack([p.sum(0).abs() for p in terms.split(rows)])
        reach = 2 * limit + torch.finfo(t.dtype).eps * want.abs()
        assert (lost.flatten(1) > reach.flatten()).any(1).all()
