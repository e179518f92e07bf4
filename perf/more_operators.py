"""What a model's attention layer does around a paged 4-bit cache, as cases that can be timed and checked.

Three operators, one layer each time:

``rotate``  the new tokens' queries and keys are normalised head by head (or not),
            rotated by their positions, and the keys and values quantised into
            their slots; read back as the cache holds them.
``scores``  attention whose scores are capped, or get a bias of distance, and whose
            rows see a window, or a prefix that is open to all of them: decode
            steps, prompts, and batches that mix them.
``shared``  attention of a batch whose requests continue one of a few long
            prefixes that the cache holds once.

Sizes are those of the package's benchmark and tests (32 query / 8 KV heads of 128
dims, 16 / 4 of 64; 509 to 131072 tokens; batches of 1 to 256) and odd ones around
them; pages of 16 to 128 tokens, groups of 32 to 128 dims.

A page holds, for each KV head (P tokens, D dims, G = D / group groups):
  k_codes int32 [P][D/8]    dim 8w+j of a token at bit 4*(j//2) + 16*(j%2) of word w
  v_codes int32 [P/8][D]    token 8w+j at that bit of word [w][d]
  k_meta, v_meta [G][P][2]  scale and zero of a token's group, in the cache's type
"""

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 1 << 25      # elements quantised at a time
PAD = 5              # rows behind the last request in a padded batch
EPS = 1e-6


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def _case(name, kind, shape, b, t, new, hq=32, hkv=8, d=128, group=64, page=64, dtype="fp16",
          pad=False, norm=False, rdim=0, neighbours=False, cap=0.0, slopes=False, window=0,
          prefix=0, groups=0, tail=0):
    c = dict(kind=kind, shape=shape, b=b, t=t, new=new, hq=hq, hkv=hkv, d=d, group=group,
             page=page, dtype=dtype, pad=pad)
    if kind == "rotate":
        c.update(norm=norm, rdim=rdim or d, neighbours=neighbours)
    else:
        c.update(cap=cap, slopes=slopes)
        c.update(dict(window=window, prefix=prefix) if kind == "scores" else
                 dict(groups=groups, tail=tail))
    return dict(c, name=name) if name else c


def listed():
    return [
        # one interactive request takes its next token: latency alone
        _case("rotate_step_b1_t509", "rotate", "step", 1, 509, 1),
        # a server's decode step, with norms of queries and keys
        _case("rotate_step_b256_t8192", "rotate", "step", 256, 8192, 1, page=16, dtype="bf16",
              norm=True),
        # a long prompt, with norms
        _case("rotate_prompt_t8192", "rotate", "prompt", 1, 0, 8192, page=128, norm=True),
        # prompts of odd lengths, neighbouring dims as pairs, half of the head rotated
        _case("rotate_prompts_d64_b7_t2041", "rotate", "prompt", 7, 0, 2041, hq=16, hkv=4, d=64,
              group=32, page=16, dtype="bf16", pad=True, rdim=32, neighbours=True),
        # one long-context stream with capped scores
        _case("cap_step_t32768", "scores", "step", 1, 32768, 1, cap=50.0),
        # a server batch of uneven requests whose scores fall with the distance
        _case("distance_step_b8_t32768", "scores", "step", 8, 32768, 1, page=16, dtype="bf16",
              slopes=True),
        # a layer with a window over long requests, capped
        _case("window_step_b16_t16001", "scores", "step", 16, 16001, 1, cap=30.0, window=4096),
        # a whole prompt, odd length, capped
        _case("cap_prompt_t4093", "scores", "prompt", 1, 0, 4093, cap=50.0),
        # prompts with a part that all of their rows see (an image, a question), odd lengths
        _case("prefix_prompts_d64_b3_t2041", "scores", "prompt", 3, 0, 2041, hq=16, hkv=4, d=64,
              group=32, page=32, dtype="bf16", pad=True, prefix=640),
        # four answers sampled for one question
        _case("shared_step_b4_t2041", "shared", "step", 4, 2041, 1, groups=1, tail=64),
        # a server's decode step behind one long instruction
        _case("shared_step_b64_t32768", "shared", "step", 64, 32768, 1, groups=1, tail=512,
              dtype="bf16"),
        # questions about two documents, odd lengths
        _case("shared_questions_b8_t8003_n61", "shared", "step", 8, 8003, 61, groups=2, tail=0,
              page=32, pad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv = rng.choice([(32, 8), (32, 8), (32, 8), (8, 2), (16, 2), (16, 16), (28, 4), (16, 4)])
    d, group = rng.choice([(128, 64), (128, 64), (128, 128), (128, 32), (64, 64), (64, 32)])
    kw = dict(hq=hq, hkv=hkv, d=d, group=group, page=rng.choice([16, 32, 64, 128]),
              dtype=rng.choice(["fp16", "bf16"]), pad=rng.random() < 0.3)
    kind = rng.choice(["rotate", "rotate", "scores", "scores", "scores", "shared", "shared"])
    if kind == "rotate":
        kw.update(norm=rng.random() < 0.5, neighbours=rng.random() < 0.3,
                  rdim=rng.choice([d, d, d, d // 2, d // 4, 16]))
        if rng.random() < 0.4:
            b = _log_int(rng, 1, 256)
            return _case(None, kind, "step", b, _log_int(rng, 16, min(8192, 262144 // b)),
                         rng.choice([1, 1, 4]), **kw)
        b = rng.choice([1, 2, 7])
        return _case(None, kind, "prompt", b, 0, _log_int(rng, 16, 8192 * 8 // (b * hkv)), **kw)
    kw.update(cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3)
    if kind == "shared":
        shape, b = "step", rng.choice([2, 4, 8, 16, 32, 64])
        new = rng.choice([1, 1, 1, 2, 4, _log_int(rng, 8, 128)])
        return _case(None, kind, shape, b, _log_int(rng, 200, 32768 * 8 // hkv // max(1, b * new // 64)),
                     new, groups=rng.choice([1, 1, 1, 2, 3]), tail=_log_int(rng, 1, 512), **kw)
    kw.update(window=rng.choice([0, 0, _log_int(rng, 16, 8192)]))
    shape = rng.choice(["step", "step", "prompt", "prompt", "mixed"])
    b = rng.choice([1, 1, 2, 4, 8, 16])
    if shape == "step":
        return _case(None, kind, shape, b, _log_int(rng, 16, min(131072, 262144 * 8 // (b * hkv))),
                     rng.choice([1, 1, 1, 2, 4, 7]), **kw)
    kw.update(prefix=rng.choice([0, 0, _log_int(rng, 8, 1024)]))
    if shape == "prompt":
        b = rng.choice([1, 1, 2, 3])
        return _case(None, kind, shape, b, 0, _log_int(rng, 16, 4093 // b), **kw)
    b = rng.choice([2, 4, 8])
    return _case(None, kind, shape, b, _log_int(rng, 200, 65536 // b), _log_int(rng, 16, 512), **kw)


# ------------------------------------------------------------------- inputs


def _requests(c):
    """(tokens held, tokens added) of every request: the first the longest,
    the others shorter by up to eight times (a prompt by four).  Of ``shared``
    the first ``groups`` are the prefixes, which add nothing; the others hold
    up to ``tail`` tokens of their own."""
    r = random.Random(c["b"] * 1000003 + c["t"] * 31 + c["new"])
    b, t, n = c["b"], c["t"], c["new"]
    if c["kind"] == "shared":
        g = c["groups"]
        held = [t] + [max(1, int(t * r.uniform(0.25, 1))) for _ in range(g - 1)]
        return held + [r.randint(0, c["tail"]) for _ in range(b)], [0] * g + [n] * b
    if c["shape"] == "prompt":
        return [0] * b, [n] + [max(1, int(n * r.uniform(0.25, 1))) for _ in range(b - 1)]
    held = [t] + [max(1, int(t * r.uniform(0.125, 1))) for _ in range(b - 1)]
    if c["shape"] == "mixed":
        return held, [n if i < max(1, b // 4) else 1 for i in range(b)]
    return held, [n] * b


def _parents(c):
    """The prefix that each request of ``shared`` continues; one in 16 none."""
    return [-1] * c["groups"] + [-1 if i % 16 == 9 else i % c["groups"] for i in range(c["b"])]


def _prefixes(c, new):
    """How many tokens all rows of each request see, of ``scores``."""
    return [max(0, min(c["prefix"] - 7 * i, 2 * n)) for i, n in enumerate(new)]


def _rows(c):
    return sum(_requests(c)[1]) + (PAD if c["pad"] else 0)


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(c, lengths, seed):
    """Block table of requests of these lengths over a pool in random order."""
    have = [-(-n // c["page"]) for n in lengths]
    total, width = sum(have) + 3, max(max(have), 1)
    order = torch.randperm(total, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    first = torch.tensor([0] + have, device="cuda").cumsum(0)[:-1]
    col = torch.arange(width, device="cuda")
    used = col[None, :] < torch.tensor(have, device="cuda")[:, None]
    at = (first[:, None] + col[None, :]).clamp(max=total - 1)
    return torch.where(used, order[at], torch.full_like(order[at], -1)), total


def _filled(c, n_pages, seed):
    """A pool of pages that hold tokens: anisotropic keys, unit values."""
    dt, d, g = DTYPES[c["dtype"]], c["d"], c["d"] // c["group"]
    hkv, page = c["hkv"], c["page"]
    gen = _gen(seed, 3)
    s = 0.5 + 3.5 * torch.rand((d,), generator=gen, device="cuda")
    kc = torch.empty((n_pages, hkv, page, d // 8), dtype=torch.int32, device="cuda")
    vc = torch.empty((n_pages, hkv, page // 8, d), dtype=torch.int32, device="cuda")
    km = torch.empty((n_pages, hkv, g, page, 2), dtype=dt, device="cuda")
    vm = torch.empty_like(km)
    per = max(1, CHUNK // (hkv * page * d))
    for i in range(0, n_pages, per):
        n = min(per, n_pages - i)
        k = (torch.randn((n, hkv, page, d), generator=gen, device="cuda") * s).to(dt)
        v = torch.randn((n, hkv, page, d), generator=gen, device="cuda").to(dt)
        kq, km[i:i + n] = _quantized(k, c["group"], (0, 1, 3, 2, 4))
        vq, vm[i:i + n] = _quantized(v, c["group"], (0, 1, 3, 2, 4))
        kc[i:i + n] = _packed(kq.unflatten(-1, (-1, 8)))
        vc[i:i + n] = _packed(vq.unflatten(2, (-1, 8)).transpose(3, 4))
    return s, [kc, vc, km, vm]


def prepare(case, seed):
    c = case
    held, new = _requests(c)
    dt, n = DTYPES[c["dtype"]], _rows(c)
    after = [h + x for h, x in zip(held, new)]
    table, total = _tables(c, after, seed)
    starts = torch.tensor([0] + new, device="cuda").cumsum(0)
    s, store = _filled(c, total, seed)
    gen = _gen(seed, 4)
    st = {"case": c, "rows": n, "store": store, "starts": starts.to(torch.int32)}
    if c["kind"] == "rotate":
        # slots and positions of the new tokens, as the scheduling step gives them
        tok = torch.arange(n, device="cuda")
        req = (torch.searchsorted(starts, tok, right=True) - 1).clamp(max=len(new) - 1)
        pos = torch.tensor(held, device="cuda")[req] + tok - starts[req]
        real = tok < starts[-1]
        col = torch.where(real, pos // c["page"], 0)
        slot = table[req, col].long() * c["page"] + pos % c["page"]
        st["slots"] = torch.where(real, slot, -1).to(torch.int32)
        st["positions"] = torch.where(real, pos, -1).to(torch.int32)
        # cosines and sines of the positions that a request may have
        half = c["rdim"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(max(after), device="cuda", dtype=torch.float64)[:, None] * freq
        st["rotary"] = torch.stack((angle.cos(), angle.sin()), -1).float()
        # before their norms queries and keys lean towards some dims, and some heads are larger
        shape, d = (n, c["hkv"], c["d"]), c["d"]
        size = 3.0 if c["norm"] else 1.0
        st["q"] = (torch.randn((n, c["hq"], d), generator=gen, device="cuda") * size * s).to(dt)
        st["k"] = (torch.randn(shape, generator=gen, device="cuda") * size * s).to(dt)
        st["v"] = torch.randn(shape, generator=gen, device="cuda").to(dt)
        w = 1.0 + 0.2 * torch.randn((2, d), generator=gen, device="cuda")
        st["qw"], st["kw"] = (w.to(dt) if c["norm"] else (None, None))
        return st
    st["q"] = torch.randn((n, c["hq"], c["d"]), generator=gen, device="cuda").to(dt)
    slopes = 2.0 ** (-8.0 * torch.arange(1, c["hq"] + 1, device="cuda") / c["hq"])
    st.update(table=table, lengths=_ints(after), scale=1.0 / math.sqrt(c["d"]), max_new=max(new),
              slopes=slopes if c["slopes"] else None)
    if c["kind"] == "scores":
        return dict(st, max_length=max(after), prefix=_ints(_prefixes(c, new)) if c["prefix"] else None)
    p = _parents(c)
    rows = [sum(x for x, y in zip(new, p) if y == g) for g in range(c["groups"])]
    return dict(st, parents=_ints(p), max_length=max(after[c["groups"]:]),
                max_shared=max(after[:c["groups"]]), group_rows=max(rows))


# -------------------------------------------------------------- plain forms


def _shifts():
    j = torch.arange(8, dtype=torch.int32, device="cuda")
    return 4 * (j // 2) + 16 * (j % 2)


def _packed(codes):
    """(..., 8) codes -> their int32 words."""
    return (codes.to(torch.int32) << _shifts()).sum(-1, dtype=torch.int32)


def _unpacked(words):
    """int32 words -> (..., 8) codes as float32."""
    return ((words[..., None] >> _shifts()) & 15).float()


def _quantized(x, group, order):
    """Codes of (..., D) rows, and each group's scale and zero, (..., G, 2)
    with its axes in `order`."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15.0).to(x.dtype).float()
    code = torch.round((g - lo) / torch.where(scale > 0, scale, 1.0)).clamp(0, 15)
    code = torch.where(scale > 0, code, 0.0).flatten(-2)
    meta = torch.cat((scale, lo), -1).to(x.dtype)
    return code, meta.permute(order)


def _write(place, words, real):
    """Adds to int32 words the difference to what they shall hold (each of
    the bits is written once; rows behind the requests write nothing)."""
    flat, at = place
    delta = torch.where(real, words - flat[at], 0)
    flat.index_put_((at,), delta, accumulate=True)


def _rotated(x, weight, s):
    """Rows (N, H, D) normalised and rotated, every operation in 32 bits (the
    mean square in 64: codes of values next to a border go by its last bit)."""
    c, y = s["case"], x.float()
    if weight is not None:
        mean = x.double().square().mean(-1, keepdim=True)
        y = y * (1.0 / torch.sqrt(mean + EPS)).float() * weight.float()
    turn = s["rotary"][s["positions"].long().clamp(min=0)][:, None]
    cos, sin = turn[..., 0], turn[..., 1]
    r = c["rdim"]
    if c["neighbours"]:
        a, b = y[..., :r:2], y[..., 1:r:2]
        z = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        z = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((z, y[..., r:]), -1).to(x.dtype)


def _rotate(s):
    c = s["case"]
    kc, vc, km, vm = s["store"]
    page, hkv, d, group = c["page"], c["hkv"], c["d"], c["group"]
    slot = s["slots"].long()
    real = (slot >= 0)[:, None, None]
    q = torch.where((s["positions"] >= 0)[:, None, None], _rotated(s["q"], s["qw"], s), 0.0)
    slot = slot.clamp(min=0)
    row = (slot // page)[:, None] * hkv + torch.arange(hkv, device="cuda")  # (N, H)
    off = (slot % page)[:, None, None]
    word, dim = torch.arange(d // 8, device="cuda"), torch.arange(d, device="cuda")
    grp = torch.arange(d // group, device="cuda")
    kq, kmeta = _quantized(_rotated(s["k"], s["kw"], s), group, (0, 1, 2, 3))
    vq, vmeta = _quantized(s["v"], group, (0, 1, 2, 3))
    at_k = (row[..., None] * page + off) * (d // 8) + word
    _write((kc.view(-1), at_k), _packed(kq.unflatten(-1, (-1, 8))), real)
    at_v = (row[..., None] * (page // 8) + off // 8) * d + dim
    shift = _shifts()[off % 8]
    old = (vc.view(-1)[at_v] >> shift) & 15
    delta = torch.where(real, (vq.to(torch.int32) - old) << shift, 0)
    vc.view(-1).index_put_((at_v,), delta, accumulate=True)
    at_m = (row[..., None] * (d // group) + grp) * page + off
    for meta, place in ((kmeta, km), (vmeta, vm)):
        pair = meta.contiguous().view(torch.int32)[..., 0]
        _write((place.view(torch.int32).view(-1), at_m), pair, real)
    # read back
    k = _unpacked(kc.view(-1)[at_k]).flatten(-2).unflatten(-1, (-1, group))
    v = ((vc.view(-1)[at_v] >> shift) & 15).float().unflatten(-1, (-1, group))
    out = {"q": q}
    for name, code, place in (("k", k, km), ("v", v, vm)):
        m = place.view(-1, 2)[at_m].float()
        x = (m[..., 1:] + code * m[..., :1]).flatten(-2)
        out[name] = torch.where(real, x, 0.0).to(s["k"].dtype)
    return out


def _held(s, table, longest):
    """Keys and values of the requests of these table rows, (R, H, T, D) float32."""
    c = s["case"]
    kc, vc, km, vm = s["store"]
    pages = table[:, :-(-longest // c["page"])].long().clamp(min=0)
    k = _unpacked(kc[pages]).flatten(-2)                       # (R, C, H, P, D)
    v = _unpacked(vc[pages]).transpose(-1, -2).flatten(3, 4)
    both = []
    for code, meta in ((k, km), (v, vm)):
        m = meta[pages].float().transpose(3, 4)                # (R, C, H, P, G, 2)
        x = m[..., 1:] + code.unflatten(-1, (-1, c["group"])) * m[..., :1]
        both.append(x.flatten(-2).transpose(1, 2).flatten(2, 3))
    return both


def _over(s, rows, k, v, pos, seen):
    """Maximum, sum and weighted values of the query rows (R, M) over keys
    (R, H, T, D); pos (R, M) in tokens of these keys, seen (R, M, T)."""
    c = s["case"]
    rep = c["hq"] // c["hkv"]
    q = s["q"].float()[rows]                                   # (R, M, Hq, D)
    q = q.unflatten(2, (c["hkv"], rep)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    score = score.unflatten(2, (rep, -1))                      # (R, H, rep, M, T)
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    if s["slopes"] is not None:
        far = (pos[..., None] - torch.arange(k.shape[2], device="cuda")).abs().float()
        score = score - s["slopes"].view(1, c["hkv"], rep, 1, 1) * far[:, None, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0)).flatten(2, 3)
    total = p.sum(-1, keepdim=True)
    parts = [x.unflatten(2, (rep, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
             for x in (top.flatten(2, 3), total, torch.matmul(p, v))]
    return parts                                               # (R, M, Hq, 1), same, (R, M, Hq, D)


def _attend(s):
    c = s["case"]
    table, starts, length = s["table"], s["starts"].long(), s["lengths"].long()
    n = starts[1:] - starts[:-1]
    tok = torch.arange(s["rows"], device="cuda")
    req = (torch.searchsorted(starts, tok, right=True) - 1).clamp(max=n.numel() - 1)
    at = (tok - starts[req]).clamp(max=s["max_new"] - 1)
    k, v = _held(s, table, s["max_length"])
    i = torch.arange(s["max_new"], device="cuda")
    pos = (length - n)[:, None] + i
    key = torch.arange(k.shape[2], device="cuda")
    seen = key <= pos[..., None]                               # (R, M, T)
    if c["kind"] == "scores":
        if s["prefix"] is not None:
            seen = seen | (key < s["prefix"][:, None, None])
        if c["window"]:
            seen = seen & (key > pos[..., None] - c["window"])
    seen = seen & (key < length[:, None, None])
    rows = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)
    top, total, out = (x[req, at] for x in _over(s, rows, k, v, pos, seen))
    if c["kind"] == "shared":
        # the children's rows, parent after parent
        p = torch.where(tok < starts[-1], s["parents"].long()[req], -1)
        key = torch.where(p < 0, n.numel(), p)
        order = torch.argsort(key, stable=True)
        first = torch.searchsorted(key[order], torch.arange(c["groups"], device="cuda"))
        place = torch.empty_like(order)
        place[order] = tok
        rows = order[(first[:, None] + torch.arange(s["group_rows"], device="cuda"))
                     .clamp(max=s["rows"] - 1)]
        k, v = _held(s, table[:c["groups"]], s["max_shared"])
        far = length[:c["groups"], None] + ((length - n)[req] + tok - starts[req])[rows]
        key = torch.arange(k.shape[2], device="cuda")
        seen = (key < length[:c["groups"], None])[:, None].expand(-1, rows.shape[1], -1)
        of = p.clamp(min=0)
        mine = (place - first[of]).clamp(0, s["group_rows"] - 1)
        more = [x[of, mine] for x in _over(s, rows, k, v, far, seen)]
        has = (p >= 0)[:, None, None]
        top2 = torch.where(has, more[0], -math.inf)
        high = torch.maximum(top, top2)
        high = torch.where(high > -math.inf, high, 0.0)
        a, b = torch.exp(top - high), torch.exp(top2 - high)
        total = a * total + b * torch.where(has, more[1], 0.0)
        out = a * out + b * torch.where(has, more[2], 0.0)
    out = out / torch.where(total > 0, total, 1.0)
    real = (tok < starts[-1])[:, None, None]
    return torch.where(real, out, 0.0).to(s["q"].dtype)


# ---------------------------------------------------------------- the calls


def run(state):
    s = state
    c = s["case"]
    if not own:
        return _rotate(s) if c["kind"] == "rotate" else _attend(s)
    S = _package()
    store = S.PagedKVStore(*s["store"])
    if c["kind"] == "rotate":
        q = S.append_rotated_paged(store, s["q"], s["k"], s["v"], s["slots"], s["positions"],
                                   s["rotary"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                   neighbours=c["neighbours"])
        k, v = S.read_paged(store, s["slots"])
        return {"q": q, "k": k, "v": v}
    kw = dict(max_new=s["max_new"], max_length=s["max_length"], softcap=c["cap"] or None,
              slopes=s["slopes"])
    if c["kind"] == "scores":
        kw.update(window=c["window"] or None, prefix_lengths=s["prefix"])
    else:
        kw["shared"] = S.build_shared_plan(s["parents"], s["lengths"], s["starts"], s["rows"],
                                           max_shared=s["max_shared"])
    return S.paged_attention(s["q"], store, s["table"], s["lengths"], s["starts"], s["scale"], **kw)


# ------------------------------------------------------------ what it takes


def _seen(c):
    """(tokens read, pairs of query row and token) of ``scores``, a head."""
    held, new = _requests(c)
    read = pairs = 0
    for h, n, x in zip(held, new, _prefixes(c, new) if c["prefix"] else [0] * len(new)):
        w = c["window"] or h + n
        read += h + n - max(0, h + 1 - w)
        for i in range(n):
            pairs += max(0, max(h + i + 1, min(x, h + n)) - max(0, h + i + 1 - w))
    return read, pairs


def work(case):
    c = case
    held, new = _requests(c)
    rows = sum(new)
    token = c["hkv"] * (c["d"] + 8 * (c["d"] // c["group"]))  # stored bytes of a token
    if c["kind"] == "rotate":
        raw = 2 * c["hkv"] * c["d"]
        return {"bytes": rows * (4 * c["hq"] * c["d"] + 4 * raw + token + 4 * c["rdim"] + 8),
                "flops": rows * (10 * c["hq"] + 50 * c["hkv"]) * c["d"]}
    if c["kind"] == "scores":
        read, pairs = _seen(c)
    else:
        p = _parents(c)
        read = sum(h + n for h, n in zip(held, new))
        pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new)) + \
            sum(n * held[x] for n, x in zip(new, p) if x >= 0)
    return {"bytes": read * token + 4 * rows * c["hq"] * c["d"], "flops": 4 * pairs * c["hq"] * c["d"]}


# --------------------------------------------------------------- in 64 bits


def _bits(words):
    """Codes of int32 words as a list over their eight places."""
    return [((words >> (4 * (j >> 1) + 16 * (j & 1))) & 15).double() for j in range(8)]


def _quantized64(x, group):
    """What the cache holds of (..., D) rows, in 64 bits."""
    x64 = x.double().reshape(*x.shape[:-1], -1, group)
    zero = x64.min(-1, keepdim=True).values
    step = ((x64.max(-1, keepdim=True).values - zero) / 15).to(x.dtype).double()
    code = ((x64 - zero) / step.clamp(min=1e-300)).round().clamp(0, 15)
    return (zero + code * step).reshape(x.shape)


def _rotated64(x, weight, s):
    """Rows in 64 bits, as complex numbers turned by their angles."""
    c, y = s["case"], x.double()
    if weight is not None:
        y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    r = c["rdim"]
    pairs = y[..., :r].unflatten(-1, (-1, 2) if c["neighbours"] else (2, -1))
    pairs = pairs if c["neighbours"] else pairs.transpose(-1, -2)
    turn = s["rotary"].double()[s["positions"].long().clamp(min=0)]
    z = torch.view_as_complex(pairs.contiguous()) * torch.view_as_complex(turn.contiguous())[:, None]
    z = torch.view_as_real(z)
    z = z if c["neighbours"] else z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), y[..., r:]), -1)


def _request64(s, r, kv, total):
    """Keys and values of one request and KV head, (T, D) in 64 bits."""
    c = s["case"]
    kc, vc, km, vm = s["store"]
    ids = s["table"][r, :-(-total // c["page"])].long()
    k = torch.stack(_bits(kc[ids, kv]), -1).reshape(-1, c["d"])[:total]
    v = torch.stack(_bits(vc[ids, kv]), 2).reshape(-1, c["d"])[:total]
    x = []
    for code, meta in ((k, km), (v, vm)):
        m = meta[ids, kv].double().permute(0, 2, 1, 3).reshape(-1, c["d"] // c["group"], 2)[:total]
        m = m.repeat_interleave(c["group"], 1)
        x.append(code * m[..., 0] + m[..., 1])
    return x


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["kind"] == "rotate":
        real = (s["slots"] >= 0).double()[:, None, None]
        k = _rotated64(s["k"], s["kw"], s).to(s["k"].dtype)
        return {"q": _rotated64(s["q"], s["qw"], s) * (s["positions"] >= 0).double()[:, None, None],
                "k": _quantized64(k, c["group"]) * real, "v": _quantized64(s["v"], c["group"]) * real}
    held, new = _requests(c)
    rep = c["hq"] // c["hkv"]
    out = torch.zeros((s["rows"], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    parents = _parents(c) if c["kind"] == "shared" else [-1] * len(new)
    opened = _prefixes(c, new) if c.get("prefix") else [0] * len(new)
    for kv in range(c["hkv"]):
        base = {p: _request64(s, p, kv, held[p]) for p in set(parents) if p >= 0}
        first = 0
        for r, (h, n) in enumerate(zip(held, new)):
            if n == 0:
                continue
            k, v = _request64(s, r, kv, h + n)
            before = 0
            if parents[r] >= 0:
                before = held[parents[r]]
                k, v = (torch.cat((a, b)) for a, b in zip(base[parents[r]], (k, v)))
            t = torch.arange(k.shape[0], device="cuda")[None, :]
            at = before + h + torch.arange(n, device="cuda")[:, None]
            hidden = (t > at) & (t >= opened[r])
            if c.get("window"):
                hidden = hidden | (t <= at - c["window"])
            for hq in range(kv * rep, (kv + 1) * rep):
                score = (s["q"][first:first + n, hq].double() @ k.t()) * s["scale"]
                if c["cap"]:
                    score = c["cap"] * torch.tanh(score / c["cap"])
                if s["slopes"] is not None:
                    score = score - s["slopes"][hq].double() * (at - t).abs()
                w = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[first:first + n, hq] = torch.nan_to_num(w, 0.0) @ v
            first += n
    return out
