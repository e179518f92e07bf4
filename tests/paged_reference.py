"""A plain 64-bit restatement of the paged 4-bit cache on the CPU: the layout
of its pages, the quantiser, the attention and the page bookkeeping."""

import math

import numpy as np
import torch

U16 = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def bit(j):
    return 4 * (j // 2) + 16 * (j % 2)


def quantize(x, group):
    """(codes, scale, zero) of (..., D) rows of a 16-bit type: codes exact in
    64 bits for the 16-bit scale and zero."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15.0).to(x.dtype)
    bad = ~torch.isfinite(g).all(-1) | ~torch.isfinite(scale.float())
    nan = torch.full_like(scale, math.nan)
    scale, zero = torch.where(bad, nan, scale), torch.where(bad, nan, lo.to(x.dtype))
    s, z = scale.double()[..., None], zero.double()[..., None]
    code = torch.round((g.double() - z) / torch.where(s > 0, s, 1.0)).clamp(0, 15)
    code = torch.where((s > 0) & ~bad[..., None], code, 0.0)
    return code.flatten(-2).to(torch.int64), scale, zero


def held(x, group):
    """What the cache holds of rows x, in 64 bits."""
    code, scale, zero = quantize(x, group)
    c = code.unflatten(-1, (-1, group)).double()
    return (zero.double()[..., None] + c * scale.double()[..., None]).flatten(-2)


def unpack(store):
    """Codes and (scale, zero) of every slot: k, v (slots, H, D) int64 and
    their metas (slots, H, G, 2), from the tensors on the CPU."""
    kc, vc, km, vm = (t.cpu() for t in store)
    n, h, p, w = kc.shape
    sh = torch.tensor([bit(j) for j in range(8)])
    k = ((kc.long()[..., None] >> sh) & 15).reshape(n, h, p, w * 8)
    v = ((vc.long()[..., None] >> sh) & 15).permute(0, 1, 2, 4, 3).reshape(n, h, p, w * 8)
    flat = lambda t: t.transpose(1, 2).reshape(n * p, *t.shape[1:2], *t.shape[3:])  # noqa: E731
    meta = lambda t: t.permute(0, 3, 1, 2, 4).reshape(n * p, h, t.shape[2], 2)      # noqa: E731
    return flat(k), flat(v), meta(km), meta(vm)


def values_of(codes, meta):
    """(slots, H, D) values in 64 bits."""
    c = codes.double().unflatten(-1, (meta.shape[2], -1))
    return (meta[..., 1:].double() + c * meta[..., :1].double()).flatten(-2)


def slots_of(table_row, length, page):
    pos = torch.arange(length)
    return table_row.cpu().long()[pos // page] * page + pos % page


def attend(q, store, table, lengths, starts, scale, causal=True, n_pages=None):
    """(out, tol): the attention in 64 bits and how far the kernels' roundings
    may take them from it.

    Per row: a score is s 64 (sum q (1 + c/64)) + (z - 64 s) sum q, sums of D
    exact products in float32: off by at most (D + 8) 2^-24 of the sum B of
    the terms' magnitudes (first order).  exp2 and the running maximum add
    2^-21; the sums over tokens at most one rounding a 32-token tile and 64
    more.  A relative change e of every probability moves an output by 2 e
    max|v|.  The output's own rounding is half a step of its type.  p s is
    rounded to fp16 (2^-11) and multiplied by code - 7.5, as the difference of
    two sums of 64 p s and 72 p s; more than 64 rows a KV head may take either
    that way or, where the call's sizes make a large one, have p and the value
    itself rounded, the value to at least 2^-18 of the largest of the
    request."""
    k_c, v_c, k_m, v_m = unpack(store)
    page = store[0].shape[2]
    k_all, v_all = values_of(k_c, k_m), values_of(v_c, v_m)
    n_rows, hq, d = q.shape
    hkv = k_c.shape[1]
    rep = hq // hkv
    out = torch.zeros((n_rows, hq, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    q64 = q.cpu().double()
    starts = starts.cpu().tolist()
    u = U16[q.dtype]
    for r, length in enumerate(lengths.cpu().tolist()):
        n = starts[r + 1] - starts[r]
        if n == 0 or length == 0:
            continue
        cols = table[r].cpu().long()[torch.arange(length) // page]
        real = (cols >= 0) & (cols < (n_pages or store[0].shape[0]))
        at = torch.where(real, cols, 0) * page + torch.arange(length) % page
        pos = torch.arange(length)
        for h in range(hkv):
            k, v = k_all[at, h], v_all[at, h]
            kt = k_m[at, h].double().repeat_interleave(d // k_m.shape[2], 1)
            kmag = kt[..., 0] * (64 + k_c[at, h]) + (kt[..., 1] - 64 * kt[..., 0]).abs()
            vt = v_m[at, h].double().repeat_interleave(d // v_m.shape[2], 1)
            middle = vt[..., 0] * (v_c[at, h] - 7.5).abs()
            largest = v.abs().nan_to_num(0.0).amax(0)
            for i in range(n):
                row = starts[r] + i
                see = real & (pos <= length - n + i) if causal else real
                if not bool(see.any()):
                    continue
                qr = q64[row, h * rep:(h + 1) * rep]
                s = (qr @ k[see].t()) * scale
                p = torch.softmax(s, -1)
                o = p @ v[see]
                out[row, h * rep:(h + 1) * rep] = o
                b = ((qr.abs() @ kmag[see].t()) * scale).amax(-1, keepdim=True)
                e = (d + 8) * 2.0 ** -24 * b + 2.0 ** -21 + (length / 32 + 64) * 2.0 ** -24
                vmax = (vt[..., 0] * v_c[at, h] + vt[..., 1].abs())[see].amax(0)
                half = 2.0 ** -11 * (p @ middle[see]) + \
                    (length / 32 + 64) * 2.0 ** -24 * 152 * (p @ vt[see][..., 0])
                if n * rep > 64:  # (either kernel's, as the call's size and hints decide)
                    half = torch.maximum(
                        half, 2.001 * 2.0 ** -11 * (p @ v[see].abs()) + 2.0 ** -18 * largest)
                tol[row, h * rep:(h + 1) * rep] = u * o.abs() + half + 2 * e * vmax + \
                    2.0 ** -24 * (1 if q.dtype == torch.float16 else 2.0 ** -100)
    return out, tol


class Pages:
    """The page bookkeeping of a step, one page at a time."""

    def __init__(self, page, width, free):
        self.page, self.width = page, width
        self.free = list(free)
        self.rows, self.lengths = [], []

    def add(self):
        self.rows.append([])
        self.lengths.append(0)

    def step(self, new):
        """Packed (slots, positions) of the new tokens."""
        need = [-(-(n + x) // self.page) for n, x in zip(self.lengths, new)]
        for row, want in zip(self.rows, need):
            self.free += row[want:]
            del row[want:]
        for row, want in zip(self.rows, need):
            while len(row) < want:
                row.append(self.free.pop())
        slots, positions = [], []
        for r, x in enumerate(new):
            for pos in range(self.lengths[r], self.lengths[r] + max(0, x)):
                slots.append(self.rows[r][pos // self.page] * self.page + pos % self.page)
                positions.append(pos)
            self.lengths[r] += x
        return np.array(slots, np.int64), np.array(positions, np.int64)


def attend_l2(q, store, table, lengths, starts, scale, causal=True):
    """(out, bound): the attention in 64 bits and, per row and query head, how
    far in L2 the kernels' roundings take it: for ordinary inputs, whose
    roundings' signs are as good as independent.  ``attend`` adds the largest
    of every error up and lets half an output pass where many tokens average;
    here each enters by its square, at its largest (true ones have a third of
    that in the mean, so a right result lies near 0.6 of the bound):

    - the output's rounding, u |o|;
    - of token t, p 2^-11 times s |c - 7.5| (p s rounded) or 2 |v| (p and v);
    - a score's error e, p e |v - o|: sqrt(D) additions' roundings of 2^-24 of
      sums that are around 80 s |q| (codes enter as 64 + c), and 2^-22 more;
    - sums over the tokens, sqrt(T / 32 + 64) roundings of 2^-24 of 160 sum(p s)."""
    k_c, v_c, k_m, v_m = unpack(store)
    page = store[0].shape[2]
    k_all, v_all = values_of(k_c, k_m), values_of(v_c, v_m)
    n_rows, hq, d = q.shape
    rep = hq // k_c.shape[1]
    out = torch.zeros((n_rows, hq, d), dtype=torch.float64)
    bound = torch.zeros((n_rows, hq), dtype=torch.float64)
    q64, starts, u = q.cpu().double(), starts.cpu().tolist(), U16[q.dtype]
    for r, length in enumerate(lengths.cpu().tolist()):
        n = starts[r + 1] - starts[r]
        if n == 0 or length == 0:
            continue
        at = slots_of(table[r], length, page)
        pos = torch.arange(length)
        for h in range(k_c.shape[1]):
            k, v, group = k_all[at, h], v_all[at, h], d // k_m.shape[2]
            ks = k_m[at, h, :, 0].double()
            vs = v_m[at, h, :, 0].double().repeat_interleave(group, 1)
            token = torch.maximum(vs * (v_c[at, h] - 7.5).abs(), 2.002 * v.abs()) * 2.0 ** -11
            for i in range(n):
                rows = slice(h * rep, (h + 1) * rep)
                qr = q64[starts[r] + i, rows]
                see = pos <= length - n + i if causal else pos >= 0
                if not bool(see.any()):
                    continue
                p = torch.softmax((qr @ k[see].t()) * scale, -1)
                o = p @ v[see]
                qg = qr.unflatten(-1, (-1, group)).norm(dim=-1)
                e = 2.0 ** -24 * d ** 0.5 * 80 * abs(scale) * (qg @ ks[see].t()) + 2.0 ** -22
                sums = 2.0 ** -24 * (length / 32 + 64) ** 0.5 * 160 * (p @ vs[see])
                vo = (v[see][None] - o[:, None]).square().sum(-1)
                square = (u * o).square().sum(-1) + p.square() @ token[see].square().sum(-1) + \
                    (p * e).square().mul(vo).sum(-1) + sums.square().sum(-1)
                out[starts[r] + i, rows], bound[starts[r] + i, rows] = o, square.sqrt()
    return out, bound


def within_l2(got, want, bound):
    """Whether every row and head of ``got`` lies within the bound."""
    return bool(((got.cpu().double() - want).norm(dim=-1) <= bound).all())
