"""A plain 64-bit restatement of the paged attention's other scores and masks,
and of requests that continue others, with what the kernels' roundings may
cost."""

import math

import torch
from paged_reference import U16, bit


def values(store):
    """(slots, H, D) codes and (slots, H, D) scales and zeros of keys, then of
    values, in 64 bits."""
    kc, vc, km, vm = store
    n, h, p, w = kc.shape
    sh = torch.tensor([bit(j) for j in range(8)], device=kc.device)
    k = ((kc.long()[..., None] >> sh) & 15).reshape(n, h, p, w * 8)
    v = ((vc.long()[..., None] >> sh) & 15).permute(0, 1, 2, 4, 3).reshape(n, h, p, w * 8)
    out = []
    for code, meta in ((k, km), (v, vm)):
        m = meta.double().repeat_interleave(w * 8 // meta.shape[2], 2)  # (n, h, D, p, 2)
        m = m.permute(4, 0, 3, 1, 2).reshape(2, n * p, h, w * 8)
        out.append((code.transpose(1, 2).reshape(n * p, h, w * 8).double(), m[0], m[1]))
    return out


def attend(q, store, table, lengths, starts, scale, causal=True, softcap=None, slopes=None,
           window=None, prefix=None, parents=None):
    """(out, tol, l2): the attention in 64 bits; per element the sum of every
    rounding's largest effect; per row and head the L2 norm of the effects,
    each by its square (for ordinary inputs, whose roundings' signs are as
    good as independent).

    A product s = scale q.k is off by (D + 8) 2^-24 of its terms' magnitudes
    (their sum is around 80 steps of a code), sqrt(D) of them in the mean; exp2
    and the running maximum by 2^-21 more.  A cap adds 2^-21 of the largest
    product or of the cap, a bias 2^-22 of itself and of the score.
    Probabilities times scales are rounded to fp16 (2^-11 of p s (code - 7.5)),
    or probabilities and values (2^-11 each), whichever kernel takes the rows;
    sums take a rounding a 32-token tile and some 64 more; the join of shared
    and own tokens 2^-21 of either.  Outputs are rounded to their type."""
    (k_c, k_s, k_z), (v_c, v_s, v_z) = values(store)
    page, dev = store[0].shape[2], q.device
    n_rows, hq, d = q.shape
    hkv = k_c.shape[1]
    rep = hq // hkv
    n_pages = store[0].shape[0]
    out = torch.zeros((n_rows, hq, d), dtype=torch.float64, device=dev)
    tol, l2 = torch.zeros_like(out), torch.zeros((n_rows, hq), dtype=torch.float64, device=dev)
    starts, lens, u = starts.cpu().tolist(), lengths.cpu().tolist(), U16[q.dtype]
    held = [max(0, min(x, table.shape[1] * page)) for x in lens]

    def tokens(r):
        pos = torch.arange(held[r], device=dev)
        cols = table[r].long()[pos // page]
        real = (cols >= 0) & (cols < n_pages)
        return torch.where(real, cols, 0) * page + pos % page, real

    for r, length in enumerate(held):
        first, n = starts[r], min(starts[r + 1], n_rows) - starts[r]
        if n <= 0 or first < 0:
            continue
        at, real = tokens(r)
        before, p = 0, -1 if parents is None else parents[r]
        if 0 <= p < len(held) and p != r:
            pat, preal = tokens(p)
            at, real, before = torch.cat((pat, at)), torch.cat((preal, real)), held[p]
        total = at.numel()
        if total == 0:
            continue
        t = torch.arange(total, device=dev)
        own = length - (starts[r + 1] - first) + torch.arange(n, device=dev)
        pos = (before + own)[:, None]
        see = (t < before) | (t <= pos) if causal else torch.ones((n, total), dtype=torch.bool, device=dev)
        if prefix is not None and causal:
            see = see | (t < min(max(0, int(prefix[r])), length))
        if window is not None:
            see = see & (t > pos.clamp(min=-1) - window)
        see = (see & real)[:, None, :].expand(n, rep, total)
        row = slice(first, first + n)
        for h in range(hkv):
            heads = slice(h * rep, (h + 1) * rep)
            qr = q[row, heads].double().reshape(n * rep, d)
            kh = k_z[at, h] + k_c[at, h] * k_s[at, h]
            s = (qr @ kh.t()).view(n, rep, total) * scale
            kmag = k_s[at, h] * (64 + k_c[at, h]) + (k_z[at, h] - 64 * k_s[at, h]).abs()
            terms = (qr.abs() @ kmag.t()).view(n, rep, total) * abs(scale)
            group = d // store[2].shape[2]
            mean = (qr.unflatten(1, (-1, group)).norm(dim=-1) @ k_s[at, h][:, ::group].t()).view(n, rep, total)
            e_max = (d + 8) * 2.0 ** -24 * terms + 2.0 ** -21
            e_l2 = 2.0 ** -24 * d ** 0.5 * 80 * abs(scale) * mean + 2.0 ** -22
            if softcap is not None:
                most = s.masked_fill(~see, 0.0).abs().amax(-1, keepdim=True)
                off = 2.0 ** -21 * torch.clamp(most, max=softcap)
                e_max, e_l2 = e_max + off, e_l2 + off
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                bias = slopes[heads].double().view(1, rep, 1) * (pos[:, None] - t).abs()
                off = 2.0 ** -22 * (bias.masked_fill(~see, 0.0).abs() + s.abs())
                e_max, e_l2, s = e_max + off, e_l2 + off, s - bias
            any_ = see.any(-1)
            s = s.masked_fill(~see, -math.inf)
            p_ = torch.softmax(s, -1).masked_fill(~any_[..., None], 0.0)
            e_max, e_l2 = (x.masked_fill(~see, 0.0) for x in (e_max, e_l2))
            vh, vs = v_z[at, h] + v_c[at, h] * v_s[at, h], v_s[at, h]
            seen_any = see.any(0).any(0)
            vh, vs = (torch.where(seen_any[:, None], x, 0.0) for x in (vh, vs))
            half = torch.where(seen_any[:, None], (vs * (v_c[at, h] - 7.5).abs()), 0.0)
            o = p_ @ vh
            sums = (total / 32 + 128) * 2.0 ** -24
            # probabilities are relative to their sum: a change of all alike is none
            e_row = (2 * (e_max * (p_ > 0)).amax(-1) + sums + 2.0 ** -21)[..., None]
            vmax = torch.where(see[..., None], (vs * v_c[at, h] + v_z[at, h].abs())[None, None], 0.0).amax(2) \
                if n * rep * total * d <= 1 << 26 else (vs * v_c[at, h] + v_z[at, h].abs()).amax(0)
            largest = vh.nan_to_num(0.0).abs().amax(0)
            each = torch.maximum(2.0 ** -11 * (p_ @ half) + sums * 152 * (p_ @ vs),
                                 2.001 * 2.0 ** -11 * (p_ @ vh.abs()) + 2.0 ** -18 * largest)
            tiny = 2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -120
            out[row, heads] = o
            tol[row, heads] = torch.where(any_[..., None], u * o.abs() + each + 2 * e_row * vmax + tiny, 0.0)
            token = torch.maximum(half, 2.002 * vh.abs()).square().sum(-1) * 2.0 ** -22
            spread = vh.square().sum(-1) - 2 * (o @ vh.t()) + o.square().sum(-1, keepdim=True)
            square = (u * o).square().sum(-1) + p_.square() @ token + \
                ((p_ * e_l2).square() * spread.clamp(min=0)).sum(-1) + \
                (2.0 ** -24 * (total / 32 + 64) ** 0.5 * 160 * (p_ @ vs)).square().sum(-1) + \
                (2.0 ** -21 * o).square().sum(-1)
            l2[row, heads] = square.sqrt()
    return out, tol, l2


def check(got, want, ordinary=True):
    """Whether ``got`` is within the bounds of ``attend``; a message if not."""
    out, tol, l2 = want
    d = got.double() - out
    far = (d.abs() > tol) & ~(got.isnan() & out.isnan()) & ~(got.double() == out)
    if bool(far.any()):
        i = int(far.flatten().nonzero()[0])
        return f"{int(far.sum())} elements off, one {d.flatten()[i]:.3g} of {tol.flatten()[i]:.3g}"
    if ordinary:
        norm = d.norm(dim=-1)
        if bool((norm > l2).any()):
            worst = (norm / l2.clamp(min=1e-300)).max()
            return f"{int((norm > l2).sum())} rows off in L2, up to {worst:.3g} of the bound"
    return ""
